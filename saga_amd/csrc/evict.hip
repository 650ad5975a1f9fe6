// What keeps a cache short: the softmax weight that every cached position gathers over a step's
// query heads, and the eviction of the positions that gathered least.
#include <algorithm>

#include "fp8.cuh"
#include "kernels.h"
#include "select.cuh"

namespace saga {

// ---- weights per position ----

// Weights of CH positions of one (batch row, group of query heads): w (+)= sum_h exp(x_h - M_h) / l_h,
// where M_h and l_h come from the softmax's partial (reference, sum) pairs.  A head without a
// finite sum (no position, a NaN score) adds nothing.  The heads of a position are added by one
// thread in their order.  Reads the scores (4 bytes a head and position) and writes 4 bytes a
// group and position; every block joins its heads' partials itself (a launch less).
constexpr int kWeightHeads = 64;  // heads whose (M, 1 / l) are held at a time

template <int PER>
__global__ void __launch_bounds__(256) attention_weights_kernel(WeightsParams p) {
  __shared__ float fm[kWeightHeads], fr[kWeightHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nchunk = (p.L + 256 * PER - 1) / (256 * PER);
  const int row = blockIdx.x / nchunk, chunk = blockIdx.x - row * nchunk;
  const int bi = row / p.G, gi = row - bi * p.G, gq = p.q_h / p.G;
  int Leff = p.L;
  if (p.kv_len) Leff = min(Leff, max(p.kv_len[bi], 0));
  const int pos0 = chunk * 256 * PER;
  float* w = p.w + bi * p.w_sb + gi * p.w_sg;
  if (pos0 >= Leff) {
    if (!p.add) {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (pos0 + k * 256 + tid < p.L) w[pos0 + k * 256 + tid] = 0.f;
    }
    return;
  }
  float acc[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = 0.f;
  for (int hb = 0; hb < gq; hb += kWeightHeads) {
    const int n = min(gq - hb, kWeightHeads);
    const int64_t r0 = static_cast<int64_t>(bi) * p.q_h + gi * gq + hb;
    if (hb) __syncthreads();
    for (int i = wave; i < n; i += 4) {
      const int64_t base = (r0 + i) * p.nparts;
      float m = kNegInf;
      for (int q = lane; q < p.nparts; q += 64) m = fmaxf(m, p.pm[(base + q) * p.pstride]);
      m = wave_max(m);
      float l = 0.f;
      for (int q = lane; q < p.nparts; q += 64) {
        const float pm = p.pm[(base + q) * p.pstride], ps = p.ps[(base + q) * p.pstride];
        l += pm == kNegInf ? ps : ps * __expf(pm - m);  // (an empty part holds (-inf, 0), one of NaN scores a NaN sum)
      }
      l = wave_sum(l);
      if (lane == 0) {
        const bool some = l > 0.f && l < __builtin_inff();
        fm[i] = some ? m : 0.f;
        fr[i] = some ? 1.f / l : 0.f;
      }
    }
    __syncthreads();
    const float* x = p.scores + r0 * p.s_ld + pos0 + tid;
    for (int i = 0; i < n; ++i) {
      const float m = fm[i], r = fr[i];
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (r > 0.f && pos0 + k * 256 + tid < Leff) acc[k] += __expf(x[i * p.s_ld + k * 256] - m) * r;
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int pos = pos0 + k * 256 + tid;
    if (pos < Leff) w[pos] = p.add ? w[pos] + acc[k] : acc[k];
    else if (pos < p.L && !p.add) w[pos] = 0.f;
  }
}

hipError_t launch_attention_weights(const WeightsParams& p, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.b) * p.G;
  const int per = rows * ((p.L + 1023) / 1024) >= 256 ? 4 : 1;
  const int64_t blocks = rows * ((p.L + 256LL * per - 1) / (256 * per));
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  if (per == 4) hipLaunchKernelGGL(attention_weights_kernel<4>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(attention_weights_kernel<1>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
  return hipGetLastError();
}

// ---- eviction ----
//
// Of n = kv_len positions `keep` stay: the last `recent`, and the H = keep - recent largest weights
// of the others.  A large one below H stays where it is, the gaps below H take the large ones
// above in order, the last `recent` follow at H: of a cache cut by a part, only that part moves,
// and in place no position above is overwritten before it is read but at the end [H, keep),
// which goes through a workspace.

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;

struct SelShared {
  int hist[2048];
  int cnt[kSelWaves];
  int sel_bin, sel_above, sel_cnt;
  int eq[kSelWaves], mov[kSelWaves], gap[kSelWaves];
};

// A weight as what it is ranked by: any NaN above all numbers, -0 as 0.
__device__ __forceinline__ float rank_value(float w) { return w == w ? w + 0.f : __uint_as_float(0x7fffffffu); }

// One block per (batch row, group): wave v holds positions [v S, (v + 1) S), lane by lane, S a
// multiple of 64, so that a position's rank in a class is a count of its wave's ballots. The
// H-th largest by radix (11, 11, 10 bits), equal ones by position.  R: passes of 64 a wave
// holds in registers, 0: reads them again (rows longer than 16 x 64 x 64).
template <int R>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
  __shared__ SelShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bi = blockIdx.x / p.G, gi = blockIdx.x - bi * p.G;
  const int n = min(max(p.kv_len[bi], 0), p.Lmax);
  const float* w = p.w + bi * p.w_sb + gi * p.w_sg;
  float* wo = p.w_out + bi * p.wo_sb + gi * p.wo_sg;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * p.keep;
  int32_t *kept = p.kept + row, *movers = p.movers + row;
  float* held = p.held_w + row;
  const int wlen = static_cast<int>(p.wo_len);
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += kSelThreads) {
      kept[j] = j < n ? j : -1;
      if (!p.in_place) wo[j] = j < n ? w[j] : 0.f;
    }
    for (int j = (p.in_place ? n : p.keep) + tid; j < wlen; j += kSelThreads) wo[j] = 0.f;
    return;
  }
  const int H = p.keep - p.recent, nc = n - p.recent;  // candidates: [0, nc), nc > H
  const int span = (nc + kSelThreads - 1) / kSelThreads * kWave, base = wave * span;
  float reg[R > 0 ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int pos = base + k * kWave + lane;
      reg[k] = k * kWave < span && pos < nc ? rank_value(w[pos]) : 0.f;
    }
  }
  // f(k, pos, value) of this lane's candidates; whole waves
  auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (k * kWave >= span) break;
        f(base + k * kWave + lane, reg[k]);
      }
    } else {
      for (int k = 0; k * kWave < span; ++k) {
        const int pos = base + k * kWave + lane;
        f(pos, pos < nc ? rank_value(w[pos]) : 0.f);
      }
    }
  };
  uint32_t T = 0xffffffffu;  // the H-th largest key
  int need = 0;              // of those equal to it, the first `need` stay
  if (H > 0) {
    need = H;
    // (positions past nc take no part: filtered by position)
    uint32_t prefix = 0;
    const int shifts[3] = {21, 10, 0}, nbits[3] = {11, 11, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int nb = 1 << nbits[pass];
      const uint32_t hmask = pass == 0 ? 0u : (0xffffffffu << (shifts[pass] + nbits[pass]));
      for (int i = tid; i < 2048; i += kSelThreads) sh.hist[i] = 0;
      lds_sync();
      each([&](int pos, float v) {
        const uint32_t key = f32_to_key(v);
        const bool in = pos < nc && (key & hmask) == prefix;
        // what never gathered anything is often many: one count for a wave
        const bool zero = in && key == 0x80000000u;
        const unsigned long long zeros = __ballot(zero);
        if (in && !zero) atomicAdd(&sh.hist[(key >> shifts[pass]) & (nb - 1)], 1);
        if (zeros && lane == 0) atomicAdd(&sh.hist[(0x80000000u >> shifts[pass]) & (nb - 1)], __popcll(zeros));
      });
      lds_sync();
      int bin, above, count;
      hist_pick<kSelThreads>(sh, nb, need, bin, above, count);
      prefix |= static_cast<uint32_t>(bin) << shifts[pass];
      need -= above;
    }
    T = prefix;
  }
  // equal ones of the waves before
  int eq = 0;
  each([&](int pos, float v) { eq += __popcll(__ballot(pos < nc && H > 0 && f32_to_key(v) == T)); });
  if (lane == 0) sh.eq[wave] = eq;
  lds_sync();
  int eq0 = 0;
  for (int i = 0; i < wave; ++i) eq0 += sh.eq[i];
  // the large ones: f(pos, value, large) in order
  const unsigned long long below = lanes_below(lane);
  auto large = [&](auto f) {
    int before = eq0;
    each([&](int pos, float v) {
      const bool in = pos < nc && H > 0;
      const uint32_t key = f32_to_key(v);
      const unsigned long long same = __ballot(in && key == T);
      const int rank = before + __popcll(same & below);
      before += __popcll(same);
      f(pos, in && (key > T || (key == T && rank < need)));
    });
  };
  int mov = 0, gap = 0;
  large([&](int pos, bool is) {
    mov += __popcll(__ballot(is && pos >= H));
    gap += __popcll(__ballot(!is && pos < H));
  });
  if (lane == 0) sh.mov[wave] = mov, sh.gap[wave] = gap;
  lds_sync();
  int mov0 = 0, gap0 = 0;
  for (int i = 0; i < wave; ++i) mov0 += sh.mov[i], gap0 += sh.gap[i];
  int at = mov0;
  large([&](int pos, bool is) {
    const unsigned long long m = __ballot(is && pos >= H);
    if (is && pos >= H) movers[at + __popcll(m & below)] = pos;
    at += __popcll(m);
  });
  __threadfence_block();
  __syncthreads();
  at = gap0;
  large([&](int pos, bool is) {
    const bool open = !is && pos < H;
    const unsigned long long m = __ballot(open);
    if (pos < H) {
      const int from = open ? movers[at + __popcll(m & below)] : pos;
      kept[pos] = from;
      held[pos] = w[from];
    }
    at += __popcll(m);
  });
  for (int j = tid; j < p.recent; j += kSelThreads) {
    kept[H + j] = nc + j;
    held[H + j] = w[nc + j];
  }
  __threadfence_block();
  __syncthreads();
  for (int j = tid; j < wlen; j += kSelThreads) wo[j] = j < p.keep ? held[j] : 0.f;
}

// Rows to their places: a block of threads per (batch row, head, S positions of the result, S a block of
// the cache's scales).  FP8: the block's scale is the largest of its rows' and a row from
// under a smaller one is rounded to it.  PHASE 0: into other tensors.  In place, two launches: 1: the blocks
// below staged0, whose rows come from at or above it or stay, and the rows of the end into the
// stage; 2: from the stage to the end.
template <int PHASE, bool FP8>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
  __shared__ int from_sh[128];
  __shared__ float scale_sh[128], red[4];
  const int tid = threadIdx.x, S = 1 << p.shift;
  const int nblk = (p.keep + S - 1) >> p.shift, staged_blk = p.staged0 >> p.shift;
  const int blocks = PHASE == 2 ? nblk - staged_blk : nblk;
  const int heads = p.rows[0].heads + p.rows[1].heads;
  int64_t id = blockIdx.x;
  const int blk = static_cast<int>(id % blocks) + (PHASE == 2 ? staged_blk : 0);
  id /= blocks;
  const int hh = static_cast<int>(id % heads), bi = static_cast<int>(id / heads);
  const bool is_v = hh >= p.rows[0].heads;
  const EvictRows& r = p.rows[is_v ? 1 : 0];
  const int h = hh - (is_v ? p.rows[0].heads : 0), gi = h / (r.heads / p.G);
  const int32_t* kept = p.kept + (static_cast<int64_t>(bi) * p.G + gi) * p.keep;
  const int j0 = blk << p.shift, count = min(S, p.keep - j0);
  const bool stage = PHASE == 1 && blk >= staged_blk;
  const int64_t nstage = p.keep - p.staged0, srow = (static_cast<int64_t>(bi) * r.heads + h) * nstage - p.staged0;  // + j
  const char* src = r.src + bi * r.s_sb + h * r.s_sh;
  char* dst = r.dst + bi * r.d_sb + h * r.d_sh;
  const float* ss = FP8 ? r.ss + bi * r.ss_sb + h * r.ss_sh : nullptr;
  float* ds = FP8 ? r.ds + bi * r.ds_sb + h * r.ds_sh : nullptr;

  float mine = 0.f;
  int any = 0;
  if (tid < count) {
    const int from = kept[j0 + tid];
    from_sh[tid] = from;
    any = from >= 0;
    if (FP8 && from >= 0) {
      mine = PHASE == 2 ? r.stage_s[srow + j0 + tid] : ss[from >> p.shift];
      scale_sh[tid] = mine;
    }
  }
  float top = 0.f, own = 0.f;
  if constexpr (FP8) {
    if (PHASE == 1 && !stage) own = ss[blk];  // (before the store below: the barrier orders them)
    top = block_max<4>(mine, red);
  }
  const bool live = __syncthreads_or(any);
  if (!live) return;
  const float inv = FP8 ? fp8_inverse(top) : 0.f;
  const int pieces = r.pieces;
  for (int e = tid; e < count * pieces; e += 256) {
    const int j = e / pieces, c = e - j * pieces, from = from_sh[j];
    if (from < 0) continue;
    if (stage) {
      *reinterpret_cast<u32x4*>(r.stage + ((srow + j0 + j) * pieces + c) * 16) = ld16(src + from * r.s_sl + 16 * c);
      if (FP8 && c == 0) r.stage_s[srow + j0 + j] = scale_sh[j];
      continue;
    }
    const float s = FP8 ? scale_sh[j] : 0.f;
    if (PHASE == 1 && from == j0 + j && (!FP8 || s == top)) continue;
    u32x4 v = ld16(PHASE == 2 ? r.stage + ((srow + j0 + j) * pieces + c) * 16 : src + from * r.s_sl + 16 * c);
    if (FP8 && s != top) v = fp8_rescaled(v, s * inv);
    *reinterpret_cast<u32x4*>(dst + (j0 + j) * r.d_sl + 16 * c) = v;
  }
  if (FP8 && tid == 0 && !stage && (PHASE != 1 || top != own)) ds[blk] = top;
}

template <bool FP8>
static void launch_evict_moves(const EvictParams& p, hipStream_t st) {
  const int64_t S = 1LL << p.shift, nblk = (p.keep + S - 1) / S;
  const int64_t rows = static_cast<int64_t>(p.B) * (p.rows[0].heads + p.rows[1].heads);
  const dim3 grid(static_cast<unsigned>(rows * nblk));
  if (!p.in_place) {
    hipLaunchKernelGGL((evict_move_kernel<0, FP8>), grid, dim3(256), 0, st, p);
    return;
  }
  hipLaunchKernelGGL((evict_move_kernel<1, FP8>), grid, dim3(256), 0, st, p);
  const int64_t rest = nblk - (p.staged0 >> p.shift);
  if (rest) hipLaunchKernelGGL((evict_move_kernel<2, FP8>), dim3(static_cast<unsigned>(rows * rest)), dim3(256), 0, st, p);
}

hipError_t launch_evict(const EvictParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.B * p.G)), block(kSelThreads);
  const int passes = (p.Lmax + kSelThreads - 1) / kSelThreads;
  if (passes <= 8) hipLaunchKernelGGL(evict_select_kernel<8>, grid, block, 0, st, p);
  else if (passes <= 32) hipLaunchKernelGGL(evict_select_kernel<32>, grid, block, 0, st, p);
  else if (passes <= 64) hipLaunchKernelGGL(evict_select_kernel<64>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, st, p);
  if (p.fp8) launch_evict_moves<true>(p, st);
  else launch_evict_moves<false>(p, st);
  return hipGetLastError();
}

}  // namespace saga
