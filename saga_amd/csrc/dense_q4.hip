// Dense decode attention over a 4-bit cache, split over the positions.
//
// A block takes one batch row, one unit of query heads (at most 16, the columns of
// every product) and one split of the positions; its waves step through 32 positions
// each and meet in LDS.  A unit is a key head with its NV whole value heads, or a run
// of heads that share both.  With the codes c as b + c (q4.cuh), b = 16 everywhere, all
// products of a step are bf16 MFMAs with 32-bit sums:
//   * x[h, j] = sum_g s_jg (q_h . c_j)_g + z_jg (sum q_h)_g: key rows straight from
//     memory as the A operand, a chain per group that starts at - sum q b;
//   * softmax with a running reference and sum in fp32: the reference moves only when
//     a score exceeds it by kSlack nats, so most steps exchange and rescale nothing;
//   * o[h, i] = sum_j (p_hj s_jg) (b + c_ji) - b sum_j p_hj s_jg + sum_j p_hj z_jg:
//     p s is split into two bf16 terms (16 bits), the first two sums are MFMAs over
//     the same terms, so that what the split loses meets c alone, the third is fp32.
//     The sums with b grow with the positions while what they leave cancels: with b 128
//     in one slot of four, an instruction less, those dims were off by 2e-4 of the
//     output over 65541 positions, the others by 3e-5 (relative norms, in the same time).
//     A lane's words of 8 positions are turned into rows of codes in registers.  A
//     column's p s are those of its own value head, whose sums alone it keeps.
// The (s, z) of a step go through wave-private LDS.  Kernel 2 joins the splits.
//
// Bound by the cache's bytes where it is large: 32 x 65541 positions, 12 / 1 / 2 heads of
// 128, groups of 32 (504 MB) 100 us, 5.0 TB/s.  A step of 32 positions is 350 VALU
// instructions and 44 MFMAs per wave for 6.9 KB (two value heads, groups of 64), about half
// of what the memory leaves time for.  Small calls are two launches and a chain of round
// trips (kernel arguments, kv_len, first step, join): 8 x 32769 positions (57 MB) 19 + 4 us,
// 1 x 4096 5.7 + 3.5; every further step per wave 1.0 us (d 64) to 2.3 (d 128, 14 MB a step).
#include <algorithm>

#include "dense_join.cuh"
#include "kernels.h"
#include "q4.cuh"

namespace saga {

// N bytes (2, 4, 8 or 16) at an address aligned to them, as dwords (2 bytes in the low half).
template <int N>
struct Bytes {
  uint32_t w[N < 4 ? 1 : N / 4];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (N == 2) w[0] = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (N == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 8) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      const u32x4 v = ld16(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    }
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int off) {
    if constexpr (N == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else if constexpr (N == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else if constexpr (N == 8) {
      const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
      w[0] = v.x, w[1] = v.y;
    } else {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (N == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (N == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
  }
};

// Two floats as a pair of bf16 numbers; a and b keep what the rounding left over.
__device__ __forceinline__ uint32_t q4_split(float& a, float& b) {
  const uint32_t w = q4_bf16_pair(a, b);
  a -= bf16_bits_to_f32(w & 0xffffu);
  b -= bf16_bits_to_f32(w >> 16);
  return w;
}

constexpr float kSlack = 8.f;  // a weight is at most e^8

// First query head of the unit `seg` of heads that share a key and a value head, cut
// at 16, and how many it holds.
__device__ __forceinline__ int q4_segment(int seg, int q_h, int g, int g_v, int& count) {
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

static int q4_segments(int q_h, int g, int g_v) {
  int n = 0;
  for (int h = 0; h < q_h; ++n) h = std::min(std::min((h / g + 1) * g, (h / g_v + 1) * g_v), h + 16);
  return n;
}

// A mask value out of the aligned word that holds it.
__device__ __forceinline__ float q4_mask_value(uint32_t word, uint32_t shift, int dt) {
  if (dt == SAGA_DTYPE_F32) return __uint_as_float(word);
  word >>= shift;
  if (dt == SAGA_DTYPE_BF16) return bf16_bits_to_f32(word & 0xffffu);
  if (dt == SAGA_DTYPE_F16) return f16_bits_to_f32(static_cast<uint16_t>(word));
  return (word & 0xffu) ? 1.f : 0.f;
}

// QT: bf16 terms of a query element (1: bf16, 2: f16).
template <int D, int G, int QT, int NV, bool MASK>
__global__ void __launch_bounds__(256, 2) dense_q4_kernel(DenseQ4Params p) {
  constexpr int NG = D / G;          // groups of a row
  constexpr int NJ = D / 32;         // MFMA steps of a row
  constexpr int NT = D / 16;         // 16-dim tiles of a row
  constexpr int SB = 4 * NG;         // bytes of a row's (s, z)
  constexpr int WROW = D + 4;
  constexpr int MERGE = 4 * 16 * (WROW + 2), SCALES = 4 * (1 + NV) * 32 * NG;  // dwords
  __shared__ __attribute__((aligned(16))) uint32_t lds[MERGE > SCALES ? MERGE : SCALES];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, s = lane >> 4;
  const int split = blockIdx.x % p.nsplit;
  const int unit = blockIdx.x / p.nsplit;
  const int bi = unit / p.nseg;
  int nh = p.g, h0 = (unit - bi * p.nseg) * p.g;
  if constexpr (NV == 1) h0 = q4_segment(unit - bi * p.nseg, p.q_h, p.g, p.g_v, nh);
  const int vh0 = h0 / p.g_v;
  int Leff = p.L;
  if (p.kv_len) Leff = min(Leff, max(p.kv_len[bi], 0));
  const int h = h0 + (col < nh ? col : 0);
  const int u_mine = NV == 1 ? 0 : h / p.g_v - vh0;

  u32x4 qraw[NJ];  // 8 dims of head `col` per MFMA step
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    qraw[j] = ld16(p.q + (bi * p.q_sb + static_cast<int64_t>(h) * p.q_sh + 32 * j + 8 * s) * 2);

  const int beg = split * p.split_len;
  const int end = min(beg + p.split_len, Leff);
  const int nstep = end > beg ? (end - beg + 31) / 32 : 0;

  // A step's rows lie within 2^31 bytes of its first: a buffer per stream and step, whose
  // size ends with the split, so that rows past it load zeros (and touch no memory).
  // Row m of key tile t is position 16 t + 4 (m % 4) + m / 4: the rows 4 s + r that a
  // lane's scores are of are then its positions 4 i + s, i = 4 t + r.
  const char* kc = p.kv.kc + bi * p.kv.kc_sb + (h0 / p.g) * p.kv.kc_sh + beg * p.kv.kc_sl;
  const char* ks = p.kv.ks + bi * p.kv.ks_sb + (h0 / p.g) * p.kv.ks_sh + beg * p.kv.ks_sl;
  const char* vc = p.kv.vc + bi * p.kv.vc_sb + vh0 * p.kv.vc_sh + beg * p.kv.vc_sl;
  const char* vs = p.kv.vs + bi * p.kv.vs_sb + vh0 * p.kv.vs_sh + beg * p.kv.vs_sl;
  const int kcl = static_cast<int>(p.kv.kc_sl), ksl = static_cast<int>(p.kv.ks_sl);
  const int vcl = static_cast<int>(p.kv.vc_sl), vsl = static_cast<int>(p.kv.vs_sl);
  const int krow = 4 * (col & 3) + (col >> 2);
  const int koff[2] = {krow * kcl + (D / 8) * s, (16 + krow) * kcl + (D / 8) * s};
  const int ksoff = (lane >> 1) * ksl + (SB / 2) * (lane & 1), vsoff = (lane >> 1) * vsl + (SB / 2) * (lane & 1);
  int voff[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) voff[i] = (4 * i + s) * vcl + (D / 32) * col;
  char* slds = reinterpret_cast<char*>(lds + w * (1 + NV) * 32 * NG);
  const char* slds_v = slds + 32 * SB * (1 + u_mine);
  const u32x4 minus16 = {0xc180c180u, 0xc180c180u, 0xc180c180u, 0xc180c180u};
  const Q4Const qc;

  struct Step {
    Bytes<D / 8> k[2];
    Bytes<D / 32> v[NV][8];
    Bytes<SB / 2> sk, sv[NV];
    uint32_t m[MASK ? 8 : 1];
  };
  // The mask of this lane's positions, of any type: the aligned word that holds a value, and
  // one shift for all (positions 4 apart are whole words apart), so that a step's loads are
  // one run without branches (a load under a branch is waited for at the join).  A batch
  // row's mask lies within 2^31 bytes.
  const int mes = p.mask_dt == SAGA_DTYPE_F32 ? 4 : p.mask_dt == SAGA_DTYPE_BOOL ? 1 : 2;
  const uint32_t mstep = static_cast<uint32_t>(p.m_sl) * mes;
  const uint64_t maddr = reinterpret_cast<uint64_t>(p.mask) + bi * p.m_sb * mes;
  const int mbytes = MASK ? static_cast<int>(maddr & 3) + static_cast<int>((p.q_h - 1) * p.m_sh + (p.L - 1) * p.m_sl + 1) * mes : 0;
  const uint32_t moff = static_cast<uint32_t>(maddr & 3) + static_cast<uint32_t>(h * p.m_sh) * mes + s * mstep;
  const uint32_t mshift = 8 * (moff & 3);
  auto load_step = [&](Step& r, int it) {
    const int c0 = 32 * it, rows = min(max(end - beg - c0, 0), 32);  // from beg
    auto buffer = [&](const char* base, int64_t stride, int row) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + c0 * stride), 0,
                                               rows ? (rows - 1) * static_cast<int>(stride) + row : 0, 0x00027000);
    };
    const auto kb = buffer(kc, p.kv.kc_sl, D / 2), ksb = buffer(ks, p.kv.ks_sl, SB);
#pragma unroll
    for (int t = 0; t < 2; ++t) r.k[t].load(kb, koff[t]);
    r.sk.load(ksb, ksoff);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      r.sv[u].load(buffer(vs + u * p.kv.vs_sh, p.kv.vs_sl, SB), vsoff);
      const auto vb = buffer(vc + u * p.kv.vc_sh, p.kv.vc_sl, D / 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[u][i].load(vb, voff[i]);
    }
    if constexpr (MASK) {
      const int64_t at = static_cast<int64_t>(beg + c0) * mstep, left = ((mbytes + 3) & ~3) - at;
      const auto mb = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>((maddr & ~uint64_t{3}) + at), 0,
                                                        left > 0 ? static_cast<int>(left) : 0, 0x00027000);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.m[i] = __builtin_amdgcn_raw_buffer_load_b32(mb, (moff + 4 * i * mstep) & ~3u, 0, 0);
    }
  };

  // the first step's loads are in flight under the query's work, the next one's under a step's
  Step ra, rb;
  load_step(ra, w);
  __builtin_amdgcn_sched_barrier(0);

  // query fragments: slots (2 k, 2 k + 1) of step j are dims 32 j + 8 s + (k, k + 4)
  u32x4 qf[NJ][QT];
  float qs[NG];   // sums over the groups, for head `col`
  f32x4 qb[NG];   // - b of them, in every row of a tile
  {
#pragma unroll
    for (int g = 0; g < NG; ++g) qs[g] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float f[8];
      if constexpr (QT == 1) unpack16<SAGA_DTYPE_BF16>(qraw[j], f);
      else unpack16<SAGA_DTYPE_F16>(qraw[j], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) qs[j * 32 / G] += f[e];
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) qf[j][t][k] = q4_split(f[k], f[k + 4]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      qs[g] += __shfl_xor(qs[g], 16);
      qs[g] += __shfl_xor(qs[g], 32);
      const float b = -16.f * qs[g];
      qb[g] = f32x4{b, b, b, b};
    }
  }

  f32x4 o[NV][NT], corr[NG];
  float zo[NG];
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < NT; ++e) o[u][e] = zero;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    corr[g] = zero;
    zo[g] = 0.f;
  }
  float m_run = kNegInf, l_run = 0.f;  // the reference of head `col`; the sum of this lane's positions

  auto use_step = [&](Step& r, int it) {
    const int c0 = beg + 32 * it;
    r.sk.store(slds + (lane >> 1) * SB + (SB / 2) * (lane & 1));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      r.sv[u].store(slds + 32 * SB * (1 + u) + (lane >> 1) * SB + (SB / 2) * (lane & 1));
    }
    wave_sync();  // (a wave's scales are private to it)
    float x[8];  // positions c0 + 4 i + s
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 dg[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        dg[g] = qb[g];
#pragma unroll
        for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
          const u32x4 a = q4_frag16(r.k[t].w[j], qc);
#pragma unroll
          for (int q = 0; q < QT; ++q) dg[g] = mfma_16b<SAGA_DTYPE_BF16>(a, qf[j][q], dg[g]);
        }
      }
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const int i = 4 * t + rr;
        Bytes<SB> sz;
        sz.load(slds + (4 * i + s) * SB);
        float v = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
          v = __builtin_fmaf(q4_lo(sz.w[g]), dg[g][rr], __builtin_fmaf(q4_hi(sz.w[g]), qs[g], v));
        x[i] = v * p.scale;
      }
    }
    if constexpr (MASK) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = x[i] + q4_mask_value(r.m[i], mshift, p.mask_dt);
    }
    if (c0 + 32 > end) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + 4 * i + s >= end) x[i] = kNegInf;
    }
    float mt = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, x[i]);
    if (__any(mt > m_run + kSlack)) {  // (from -inf on: any score)
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = fmaxf(mt, __shfl_xor(mt, 32));
      const float m_new = fmaxf(m_run, mt);
      const float alpha = m_run == kNegInf ? (m_new == kNegInf ? 1.f : 0.f) : __expf(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < NT; ++e) o[u][e] *= alpha;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        corr[g] *= alpha;
        zo[g] *= alpha;
      }
    }
    const float m_ref = m_run == kNegInf ? 0.f : m_run;  // (no score yet: weights of 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __expf(x[i] - m_ref);
      l_run += x[i];
    }
    u32x4 pf[NG][2];
    {
      float pv[NG][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        Bytes<SB> sz;
        sz.load(slds_v + (4 * i + s) * SB);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pv[g][i] = __builtin_fmaf(q4_lo(sz.w[g]), x[i], 0.f);  // reads the f16 as it is
          zo[g] = __builtin_fmaf(q4_hi(sz.w[g]), x[i], zo[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) pf[g][k][i] = q4_split(pv[g][2 * i], pv[g][2 * i + 1]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int k = 0; k < 2; ++k) corr[g] = mfma_16b<SAGA_DTYPE_BF16>(minus16, pf[g][k], corr[g]);
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int hv = 0; hv < NT / 4; ++hv) {  // halves of a unit of nibbles: dims 64 hv ..
        uint32_t two[4];  // codes of positions 2 k, 2 k + 1
#pragma unroll
        for (int k = 0; k < 4; ++k)
          two[k] = __builtin_amdgcn_perm(r.v[u][2 * k + 1].w[0], r.v[u][2 * k].w[0], hv == 0 ? 0x05040100u : 0x07060302u);
        auto tile = [&](int e, const u32x4& a) {
#pragma unroll
          for (int k = 0; k < 2; ++k) o[u][e] = mfma_16b<SAGA_DTYPE_BF16>(a, pf[16 * e / G][k], o[u][e]);
        };
        tile(4 * hv + 0, u32x4{q4_pair16<0>(two[0], qc), q4_pair16<0>(two[1], qc), q4_pair16<0>(two[2], qc), q4_pair16<0>(two[3], qc)});
        tile(4 * hv + 1, u32x4{q4_pair<1>(two[0], qc), q4_pair<1>(two[1], qc), q4_pair<1>(two[2], qc), q4_pair<1>(two[3], qc)});
        tile(4 * hv + 2, u32x4{q4_pair<2>(two[0], qc), q4_pair<2>(two[1], qc), q4_pair<2>(two[2], qc), q4_pair<2>(two[3], qc)});
        tile(4 * hv + 3, u32x4{q4_pair<3>(two[0], qc), q4_pair<3>(two[1], qc), q4_pair<3>(two[2], qc), q4_pair<3>(two[3], qc)});
      }
    wave_sync();  // the scales are rewritten by this wave's next step
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

  __syncthreads();  // every wave is done with its scales
  float* Wo = reinterpret_cast<float*>(lds);
  float (*Wm)[16] = reinterpret_cast<float (*)[16]>(Wo + 4 * 16 * WROW);
  float (*Wl)[16] = Wm + 4;
  // the lanes of a head hold its positions between them
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    zo[g] += __shfl_xor(zo[g], 16);
    zo[g] += __shfl_xor(zo[g], 32);
  }
  if (s == 0) {
    Wm[w][col] = m_run;
    Wl[w][col] = l_run;
  }
#pragma unroll
  for (int e = 0; e < NT; ++e) {
    f32x4 a = o[0][e];
#pragma unroll
    for (int u = 1; u < NV; ++u) a = u_mine == u ? o[u][e] : a;
    const int g = 16 * e / G;
    *reinterpret_cast<f32x4*>(Wo + (w * 16 + col) * WROW + 16 * e + 4 * s) = a + (corr[g] + zo[g]);
  }
  __syncthreads();

  // join the four waves: the split's partial, or the output when nsplit == 1
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
    if (p.nsplit == 1) {
      store_from_f32(p.out, p.out_dt, bi * p.o_sb + static_cast<int64_t>(h0 + hh) * p.o_sh + dd, q4_in_range(a / l, p.out_dt));
    } else {
      const int64_t at = (static_cast<int64_t>(bi) * p.q_h + h0 + hh) * p.nsplit + split;
      p.part[at * D + dd] = a;
      if (dd == 0) reinterpret_cast<float2*>(p.part + static_cast<int64_t>(p.b) * p.q_h * p.nsplit * D)[at] = float2{M, l};
    }
  }
}

// As many splits as keep every block resident, two per CU (a few blocks more ran after
// the others: 8 of 520 took 3 us of 26), each of at least a step per wave; up to 512
// positions in one, without a join (400 positions 6.4 - 9.9 us against 7.4 - 9.5 in a graph, and
// a launch less, 3 us, for an eager caller).  The plan is the cache's: a row filled to a part keeps
// few of its blocks busy (8 rows of 4096, 11 us in a cache of 4096 positions, 17 in 33024, 40 in
// 131072).  More units never get more splits, so a plan for b units bounds every other.
void dense_q4_plan(int64_t units, int64_t L, int64_t* nsplit, int64_t* split_len) {
  const int64_t ns = std::max<int64_t>(512 / std::max<int64_t>(units, 1), 1);
  const int64_t sl = std::max<int64_t>(((L + ns - 1) / ns + 31) / 32 * 32, L <= 512 ? 512 : 128);
  *split_len = sl;
  *nsplit = (L + sl - 1) / sl;
}

// Whether masked calls take units of NV value heads.  With four groups of each row the registers of
// two value heads spill: 8 x 30k positions, 12 / 1 / 2 heads, 41 us as two units against 62.
constexpr bool dense_q4_masked(int D, int G, int NV) { return NV == 1 || D / G < 4; }

template <int D, int G, int QT, int NV>
static void launch_dense_q4_typed(const DenseQ4Params& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.b * p.nseg * p.nsplit));
  if constexpr (dense_q4_masked(D, G, NV)) {
    if (p.mask) {
      hipLaunchKernelGGL((dense_q4_kernel<D, G, QT, NV, true>), grid, dim3(256), 0, st, p);
      return;
    }
  }
  hipLaunchKernelGGL((dense_q4_kernel<D, G, QT, NV, false>), grid, dim3(256), 0, st, p);
}

template <int D, int G, int QT>
static void launch_dense_q4_units(const DenseQ4Params& p, int nv, hipStream_t st) {
  if constexpr (D == 64) {
    if (nv == 5) return launch_dense_q4_typed<D, G, QT, 5>(p, st);
  }
  if (nv == 2) return launch_dense_q4_typed<D, G, QT, 2>(p, st);
  launch_dense_q4_typed<D, G, QT, 1>(p, st);
}

template <int D, int G>
static void launch_dense_q4_group(const DenseQ4Params& p, int nv, hipStream_t st) {
  if (p.q_dt == SAGA_DTYPE_BF16) launch_dense_q4_units<D, G, 1>(p, nv, st);
  else launch_dense_q4_units<D, G, 2>(p, nv, st);
}

hipError_t launch_dense_decode_q4(DenseQ4Params& p, hipStream_t st) {
  // A key head with its value heads in one unit reads and scores its keys once; built for
  // the decoder's layouts, 2 and (d 64) 5 value heads
  const int n_k = p.q_h / p.g;
  int nv = p.g % p.g_v == 0 && p.g <= 16 ? p.g / p.g_v : 1;
  if (nv != 2 && !(nv == 5 && p.kv.d == 64)) nv = 1;
  // (the units of five value heads spill with a mask too, 14 to 77 registers, and pay for it only with
  // groups of 32: 8 x 32768 positions, 15 / 1 / 5 heads of 64, bf16 and f16, 54 and 63 us against 47 and
  // 50 as five units, with groups of 64 28 and 38 against 41 and 45)
  if (p.mask && !dense_q4_masked(p.kv.d, p.kv.group, nv)) nv = 1;
  int64_t ns, sl;
  if (nv > 1) {
    // (not where that leaves most CUs without a block)
    dense_q4_plan(static_cast<int64_t>(p.b) * n_k, p.L, &ns, &sl);
    if (p.b * n_k * ns < 128) nv = 1;
  }
  p.nseg = nv > 1 ? n_k : q4_segments(p.q_h, p.g, p.g_v);
  dense_q4_plan(static_cast<int64_t>(p.b) * p.nseg, p.L, &ns, &sl);
  p.nsplit = static_cast<int32_t>(ns);
  p.split_len = static_cast<int32_t>(sl);
  if (p.b * p.nseg * ns >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  if (p.kv.d == 128) {
    if (p.kv.group == 32) launch_dense_q4_group<128, 32>(p, nv, st);
    else launch_dense_q4_group<128, 64>(p, nv, st);
    if (ns > 1) launch_dense_join<128>(p, st);
  } else {
    if (p.kv.group == 32) launch_dense_q4_group<64, 32>(p, nv, st);
    else launch_dense_q4_group<64, 64>(p, nv, st);
    if (ns > 1) launch_dense_join<64>(p, st);
  }
  return hipGetLastError();
}

}  // namespace saga
