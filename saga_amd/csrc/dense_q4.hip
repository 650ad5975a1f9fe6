// Dense decode attention over a 4-bit cache, split over the positions.
//
// A block takes one batch row, one run of query heads that share a key head and
// a value head (at most 16, the columns of every product) and one split of the
// positions; its waves step through 32 positions each and meet in LDS.  With the
// codes c as 16 + c (q4.cuh), all products of a step are bf16 MFMAs with 32-bit
// sums:
//   * x[h, j] = sum_g s_jg (q_h . (16 + c_j))_g + (z_jg - 16 s_jg) (sum q_h)_g:
//     key rows straight from memory as the A operand, one chain per group;
//   * softmax with a running maximum and sum, all in fp32;
//   * o[h, i] = sum_j (p_hj s_jg) (16 + c_ji) - 16 sum_j p_hj s_jg + sum_j p_hj z_jg:
//     p s is split into two bf16 terms (16 bits), the first two sums are MFMAs over
//     the same terms, so that what the split loses meets c alone, the third is fp32.
//     A lane's words of 8 positions are turned into rows of codes in registers.
// Kernel 2 joins the splits.
#include <algorithm>

#include "kernels.h"
#include "q4.cuh"

namespace saga {

// Wave-local LDS ordering: a wave's scales are private to it.
__device__ __forceinline__ void q4_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (N == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (N == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
  }
};

// Two floats as a pair of bf16 numbers; a and b keep what the rounding left over.
__device__ __forceinline__ uint32_t q4_split(float& a, float& b) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2_t));
  a -= bf16_bits_to_f32(w & 0xffffu);
  b -= bf16_bits_to_f32(w >> 16);
  return w;
}

// First query head of the unit `seg` and how many it holds: runs of one key head
// and one value head, cut at 16.
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

// QT: bf16 terms of a query element (1: bf16, 2: f16).
template <int D, int G, int QT>
__global__ void __launch_bounds__(256, 2) dense_q4_kernel(DenseQ4Params p) {
  constexpr int NG = D / G;          // groups of a row
  constexpr int NJ = D / 32;         // MFMA steps of a row
  constexpr int NT = D / 16;         // 16-dim tiles of a row
  constexpr int SB = 4 * NG;         // bytes of a row's (s, z)
  constexpr int WROW = D + 4;
  constexpr int MERGE = 4 * 16 * (WROW + 2), SCALES = 4 * 2 * 32 * NG;  // dwords
  __shared__ __attribute__((aligned(16))) uint32_t lds[MERGE > SCALES ? MERGE : SCALES];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, s = lane >> 4;
  const int split = blockIdx.x % p.nsplit;
  const int unit = blockIdx.x / p.nsplit;
  const int bi = unit / p.nseg;
  int nh;
  const int h0 = q4_segment(unit - bi * p.nseg, p.q_h, p.g, p.g_v, nh);
  int Leff = p.L;
  if (p.kv_len) Leff = min(Leff, max(p.kv_len[bi], 0));
  const int h = h0 + (col < nh ? col : 0);

  // query fragments: slots (2 k, 2 k + 1) of step j are dims 32 j + 8 s + (k, k + 4)
  u32x4 qf[NJ][QT];
  float qs[NG];  // sums over the groups, for head `col`
#pragma unroll
  for (int g = 0; g < NG; ++g) qs[g] = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const u32x4 v = ld16(p.q + (bi * p.q_sb + static_cast<int64_t>(h) * p.q_sh + 32 * j + 8 * s) * 2);
    float f[8];
    if constexpr (QT == 1) unpack16<SAGA_DTYPE_BF16>(v, f);
    else unpack16<SAGA_DTYPE_F16>(v, f);
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
  }

  const char* kc = p.kv.kc + bi * p.kv.kc_sb + (h0 / p.g) * p.kv.kc_sh + (D / 8) * s;
  const char* ks = p.kv.ks + bi * p.kv.ks_sb + (h0 / p.g) * p.kv.ks_sh + (SB / 2) * (lane & 1);
  const char* vc = p.kv.vc + bi * p.kv.vc_sb + (h0 / p.g_v) * p.kv.vc_sh + (D / 32) * col;
  const char* vs = p.kv.vs + bi * p.kv.vs_sb + (h0 / p.g_v) * p.kv.vs_sh + (SB / 2) * (lane & 1);
  // row m of key tile t is position 16 t + 4 (m % 4) + m / 4: the rows 4 s + r that a
  // lane's scores are of are then its positions 4 i + s, i = 4 t + r
  const int krow = 4 * (col & 3) + (col >> 2);
  char* slds = reinterpret_cast<char*>(lds + w * 2 * 32 * NG);
  const u32x4 minus16 = {0xc180c180u, 0xc180c180u, 0xc180c180u, 0xc180c180u};

  const int beg = split * p.split_len;
  const int end = min(beg + p.split_len, Leff);
  const int nstep = end > beg ? (end - beg + 31) / 32 : 0;

  struct Step {
    Bytes<D / 8> k[2];
    Bytes<D / 32> v[8];
    Bytes<SB / 2> sk, sv;
  };
  // positions past the range repeat its last one (their weight is 0)
  auto load_step = [&](Step& r, int c0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) r.k[t].load(kc + static_cast<int64_t>(min(c0 + 16 * t + krow, end - 1)) * p.kv.kc_sl);
    const int64_t row = min(c0 + (lane >> 1), end - 1);
    r.sk.load(ks + row * p.kv.ks_sl);
    r.sv.load(vs + row * p.kv.vs_sl);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i].load(vc + static_cast<int64_t>(min(c0 + 4 * i + s, end - 1)) * p.kv.vc_sl);
  };

  f32x4 o[NT], corr[NG];
  float zo[NG];
#pragma unroll
  for (int e = 0; e < NT; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    corr[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    zo[g] = 0.f;
  }
  float m_run = kNegInf, l_run = 0.f;

  for (int it = w; it < nstep; it += 4) {
    const int c0 = beg + 32 * it;
    Step r;
    load_step(r, c0);
    r.sk.store(slds + (lane >> 1) * SB + (SB / 2) * (lane & 1));
    r.sv.store(slds + 32 * SB + (lane >> 1) * SB + (SB / 2) * (lane & 1));
    q4_wave_sync();
    float x[8];  // positions c0 + 4 i + s
    float mt = kNegInf;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 dg[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        dg[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
          const u32x4 a = q4_frag(r.k[t].w[j]);
#pragma unroll
          for (int q = 0; q < QT; ++q) dg[g] = mfma_16b<SAGA_DTYPE_BF16>(a, qf[j][q], dg[g]);
        }
      }
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const int i = 4 * t + rr, pos = c0 + 4 * i + s;
        Bytes<SB> sz;
        sz.load(slds + (4 * i + s) * SB);
        float v = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float sc = q4_lo(sz.w[g]);
          v = __builtin_fmaf(sc, dg[g][rr], v);
          v = __builtin_fmaf(__builtin_fmaf(-16.f, sc, q4_hi(sz.w[g])), qs[g], v);
        }
        v *= p.scale;
        if (p.mask)
          v = v + load_as_f32(p.mask, p.mask_dt, bi * p.m_sb + static_cast<int64_t>(h) * p.m_sh +
                                                     static_cast<int64_t>(min(pos, p.L - 1)) * p.m_sl);
        if (pos >= end) v = kNegInf;
        x[i] = v;
        mt = fmaxf(mt, v);
      }
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16));
    mt = fmaxf(mt, __shfl_xor(mt, 32));
    const float m_new = fmaxf(m_run, mt);
    const float alpha = (m_run == kNegInf) ? (m_new == kNegInf ? 1.f : 0.f) : __expf(m_run - m_new);
    float ps = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = x[i] == kNegInf ? 0.f : __expf(x[i] - m_new);
      ps += x[i];
    }
    ps += __shfl_xor(ps, 16);
    ps += __shfl_xor(ps, 32);
    l_run = l_run * alpha + ps;
    m_run = m_new;
#pragma unroll
    for (int e = 0; e < NT; ++e) o[e] *= alpha;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      corr[g] *= alpha;
      zo[g] *= alpha;
    }
    u32x4 pf[NG][2];
    {
      float pv[NG][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        Bytes<SB> sz;
        sz.load(slds + 32 * SB + (4 * i + s) * SB);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pv[g][i] = x[i] * q4_lo(sz.w[g]);
          zo[g] = __builtin_fmaf(x[i], q4_hi(sz.w[g]), zo[g]);
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
    for (int hv = 0; hv < NT / 4; ++hv) {  // halves of a unit: dims 64 hv ..
      uint32_t two[4];  // codes of positions 2 k, 2 k + 1
#pragma unroll
      for (int k = 0; k < 4; ++k)
        two[k] = hv == 0 ? __builtin_amdgcn_perm(r.v[2 * k + 1].w[0], r.v[2 * k].w[0], 0x05040100u)
                         : __builtin_amdgcn_perm(r.v[2 * k + 1].w[0], r.v[2 * k].w[0], 0x07060302u);
      auto tile = [&](int e, const u32x4& a) {
        const int g = 16 * e / G;
#pragma unroll
        for (int k = 0; k < 2; ++k) o[e] = mfma_16b<SAGA_DTYPE_BF16>(a, pf[g][k], o[e]);
      };
      tile(4 * hv + 0, u32x4{q4_pair<0>(two[0]), q4_pair<0>(two[1]), q4_pair<0>(two[2]), q4_pair<0>(two[3])});
      tile(4 * hv + 1, u32x4{q4_pair<1>(two[0]), q4_pair<1>(two[1]), q4_pair<1>(two[2]), q4_pair<1>(two[3])});
      tile(4 * hv + 2, u32x4{q4_pair<2>(two[0]), q4_pair<2>(two[1]), q4_pair<2>(two[2]), q4_pair<2>(two[3])});
      tile(4 * hv + 3, u32x4{q4_pair<3>(two[0]), q4_pair<3>(two[1]), q4_pair<3>(two[2]), q4_pair<3>(two[3])});
    }
    q4_wave_sync();  // the scales are rewritten by this wave's next step
  }

  __syncthreads();  // every wave is done with its scales
  float* Wo = reinterpret_cast<float*>(lds);
  float (*Wm)[16] = reinterpret_cast<float (*)[16]>(Wo + 4 * 16 * WROW);
  float (*Wl)[16] = Wm + 4;
  if (s == 0) {
    Wm[w][col] = m_run;
    Wl[w][col] = l_run;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {  // the lanes of a head hold its positions between them
    zo[g] += __shfl_xor(zo[g], 16);
    zo[g] += __shfl_xor(zo[g], 32);
  }
#pragma unroll
  for (int e = 0; e < NT; ++e)
    *reinterpret_cast<f32x4*>(Wo + (w * 16 + col) * WROW + 16 * e + 4 * s) = o[e] + (corr[16 * e / G] + zo[16 * e / G]);
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
      store_from_f32(p.out, p.out_dt, bi * p.o_sb + static_cast<int64_t>(h0 + hh) * p.o_sh + dd, a / l);
    } else {
      float* part = p.part + ((static_cast<int64_t>(bi) * p.q_h + h0 + hh) * p.nsplit + split) * (2 + D);
      part[2 + dd] = a;
      if (dd == 0) {
        part[0] = M;
        part[1] = l;
      }
    }
  }
}

// Joins a head's splits: one block per (batch row, head), 8 x D threads; thread
// (grp, i) sums dim i of the splits grp, grp + 8, ..., the groups add up in a
// fixed order.
template <int D>
__global__ void __launch_bounds__(8 * D) dense_q4_join_kernel(DenseQ4Params p) {
  constexpr int NT = 8 * D;
  __shared__ float fm[1024];
  __shared__ float red[NT / kWave];
  __shared__ float og[8][D];
  const int tid = threadIdx.x, grp = tid / D, i = tid - grp * D;
  const int bi = blockIdx.x / p.q_h, h = blockIdx.x - bi * p.q_h;
  const float* base = p.part + static_cast<int64_t>(blockIdx.x) * p.nsplit * (2 + D);
  float mloc = kNegInf;
  for (int q = tid; q < p.nsplit; q += NT) {
    fm[q] = base[q * (2 + D)];
    mloc = fmaxf(mloc, fm[q]);
  }
  const float M = block_max<NT / kWave>(mloc, red);
  float lloc = 0.f;
  for (int q = tid; q < p.nsplit; q += NT) {
    const float lq = base[q * (2 + D) + 1];
    const float f = fm[q] == kNegInf ? (lq == 0.f ? 0.f : 1.f) : __expf(fm[q] - M);
    lloc += lq * f;
    fm[q] = f;
  }
  const float l = block_sum<NT / kWave>(lloc, red);  // orders the writes of fm too
  float a = 0.f;
  for (int q0 = grp; q0 < p.nsplit; q0 += 64) {
    float ov[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) ov[u] = q0 + 8 * u < p.nsplit ? base[(q0 + 8 * u) * (2 + D) + 2 + i] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (q0 + 8 * u < p.nsplit) a += ov[u] * fm[q0 + 8 * u];
  }
  og[grp][i] = a;
  __syncthreads();
  if (grp == 0) {
    float t = og[0][i];
#pragma unroll
    for (int q = 1; q < 8; ++q) t += og[q][i];
    store_from_f32(p.out, p.out_dt, bi * p.o_sb + static_cast<int64_t>(h) * p.o_sh + i, t / l);
  }
}

// About 512 blocks over b batch rows, splits of whole 32-position steps and of at
// least 64 positions; at most 1024 (the join kernel's table).
void dense_q4_plan(int64_t b, int64_t L, int64_t* nsplit, int64_t* split_len) {
  int64_t ns = std::max<int64_t>(512 / std::max<int64_t>(b, 1), 1);
  ns = std::min<int64_t>(ns, (L + 63) / 64);
  int64_t sl = (L + ns - 1) / ns;
  sl = (sl + 31) / 32 * 32;
  *split_len = sl;
  *nsplit = (L + sl - 1) / sl;
}

template <int D, int G>
static void launch_dense_q4_typed(const DenseQ4Params& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.b * p.nseg * p.nsplit));
  if (p.q_dt == SAGA_DTYPE_BF16) hipLaunchKernelGGL((dense_q4_kernel<D, G, 1>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((dense_q4_kernel<D, G, 2>), grid, dim3(256), 0, st, p);
}

hipError_t launch_dense_decode_q4(DenseQ4Params& p, hipStream_t st) {
  p.nseg = q4_segments(p.q_h, p.g, p.g_v);
  if (static_cast<int64_t>(p.b) * p.nseg * p.nsplit >= (1LL << 24)) return hipErrorInvalidValue;
  if (p.kv.d == 128) {
    if (p.kv.group == 32) launch_dense_q4_typed<128, 32>(p, st);
    else launch_dense_q4_typed<128, 64>(p, st);
    if (p.nsplit > 1) hipLaunchKernelGGL((dense_q4_join_kernel<128>), dim3(p.b * p.q_h), dim3(1024), 0, st, p);
  } else {
    if (p.kv.group == 32) launch_dense_q4_typed<64, 32>(p, st);
    else launch_dense_q4_typed<64, 64>(p, st);
    if (p.nsplit > 1) hipLaunchKernelGGL((dense_q4_join_kernel<64>), dim3(p.b * p.q_h), dim3(512), 0, st, p);
  }
  return hipGetLastError();
}

}  // namespace saga
