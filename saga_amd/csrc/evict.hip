// What keeps a cache short: the softmax weight that every cached position gathers over a step's
// query heads, and the eviction of the positions that gathered least.
#include <algorithm>

#include "fp8.cuh"
#include "kernels.h"
#include "select.cuh"

namespace saga {

// ---- weights per position ----

// w (+)= sum_h exp(x_h - M_h) / l_h of one (batch row, group of query heads), where M_h and l_h come from
// the softmax's partial (reference, sum) pairs.  A head without a finite sum (no position, a NaN
// score) adds nothing.  A thread takes 4 positions and adds their heads in order.  Every block
// joins its heads' partials itself (a launch less), under the loads of its first scores.
// Bound by the scores, 4 bytes a head and position: 32 x 65544 positions of 12 heads (109 MB)
// 22 us, 4.9 TB/s; 8 x 33024 6.3 (a position a thread: 38 and 8.9).
constexpr int kWeightHeads = 64;  // heads whose (M, 1 / l) are held at a time

__global__ void __launch_bounds__(256) attention_weights_kernel(WeightsParams p) {
  constexpr int PER = 4, TH = 4;  // positions of a thread, heads whose scores are in flight at a time
  __shared__ float fm[kWeightHeads], fr[kWeightHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nchunk = (p.L + 256 * PER - 1) / (256 * PER);
  const int row = blockIdx.x / nchunk, pos0 = (blockIdx.x - row * nchunk) * 256 * PER, pos = pos0 + tid * PER;
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

hipError_t launch_attention_weights(const WeightsParams& p, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.b) * p.G;
  const int64_t blocks = rows * ((p.L + 1023LL) / 1024);
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  hipLaunchKernelGGL(attention_weights_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
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

template <int SEG>
struct SelShared {
  uint32_t key[SEG];  // ranking keys; then, of a row of one segment, the positions that move
  int hist[2048];
  int cnt[kSelWaves];
  int sel_bin, sel_above, sel_cnt;
  int sums[3][kSelWaves];
  unsigned long long a[SEG / kWave], b[SEG / kWave];  // per chunk: masks of keys above T and equal to it, then of
  int a0[SEG / kWave], b0[SEG / kWave];               // those that move and of the gaps, and their first ones' ranks
};

// A weight as what it is ranked by: any NaN above all numbers, -0 as 0; never 0, which stands for no position.
__device__ __forceinline__ uint32_t rank_key(float w) { return f32_to_key(w == w ? w + 0.f : __uint_as_float(0x7fffffffu)); }

// The lowest `count` set bits of m.
__device__ __forceinline__ unsigned long long low_bits(unsigned long long m, int count) {
  if (count == 0) return 0ull;
  const int drop = __popcll(m) - count;
  for (int i = 0; i < drop; ++i) m &= ~(1ull << (63 - __clzll(static_cast<long long>(m))));
  return m;
}

// Bits of positions below `end` of a chunk of 64 that starts at p0.
__device__ __forceinline__ unsigned long long bits_below(int end, int p0) {
  const int n = min(max(end - p0, 0), 64);
  return n == 0 ? 0ull : ~0ull >> (64 - n);
}

// One block per (batch row, group), a segment of SEG positions' ranking keys in LDS (a row of one
// segment is read once, longer ones for every pass).  The H-th largest key by radix (11, 11, 10
// bits), equal ones by position.  What is large of a chunk of 64 positions is then one 64-bit
// mask, and thread c counts chunk c: every prefix of the selection is one scan of the block, and a
// wave places its chunks' positions with one count each.
template <int SEG>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
  __shared__ SelShared<SEG> sh;
  constexpr int CH = SEG / kWave;
  static_assert(CH <= kSelThreads && SEG % kSelThreads == 0, "a thread per chunk");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bi = blockIdx.x / p.G, gi = blockIdx.x - bi * p.G;
  const int n = min(max(p.kv_len[bi], 0), p.Lmax);
  const float* w = p.w + bi * p.w_sb + gi * p.w_sg;
  float* wo = p.w_out + bi * p.wo_sb + gi * p.wo_sg;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * p.keep;
  int32_t *kept = p.kept + row, *movers = p.movers + row;
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
  const int nseg = (nc + SEG - 1) / SEG;
  constexpr int U = 4;
  auto load = [&](int seg) {  // (a thread's own keys: no barrier is needed to count them)
    const int whole = (min(SEG, nc - seg * SEG) + kWave - 1) / kWave * kWave;  // the last chunk's end too
    for (int j0 = tid; j0 < whole; j0 += 2 * U * kSelThreads) {
      float v[2 * U];
#pragma unroll
      for (int u = 0; u < 2 * U; ++u) v[u] = w[min(seg * SEG + j0 + u * kSelThreads, nc - 1)];
#pragma unroll
      for (int u = 0; u < 2 * U; ++u)
        if (j0 + u * kSelThreads < SEG) sh.key[j0 + u * kSelThreads] = seg * SEG + j0 + u * kSelThreads < nc ? rank_key(v[u]) : 0u;
    }
  };
  // f(chunk, key) of the segment's chunks, wave by wave; keys are 0 behind nc
  auto chunks = [&](int seg, auto f) {
    const int nch = (min(SEG, nc - seg * SEG) + kWave - 1) / kWave;
    for (int c0 = wave; c0 < nch; c0 += U * kSelWaves) {
      uint32_t key[U];
#pragma unroll
      for (int u = 0; u < U; ++u) key[u] = c0 + u * kSelWaves < nch ? sh.key[(c0 + u * kSelWaves) * kWave + lane] : 0u;
#pragma unroll
      for (int u = 0; u < U; ++u) f(c0 + u * kSelWaves, key[u]);
    }
  };
  load(0);
  uint32_t T = 0xffffffffu;  // the H-th largest key
  int need = 0;              // of those equal to it, the first `need` stay
  if (H > 0) {
    constexpr uint32_t kZero = 0x80000000u;
    need = H;
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, nb = pass == 2 ? 1024 : 2048;
      const uint32_t hmask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < 2048; i += kSelThreads) sh.hist[i] = 0;
      lds_sync();
      int zeros = 0;  // weights of 0 may be many: counted by the wave (what is no position counts in the lowest bin)
      for (int seg = 0; seg < nseg; ++seg) {
        if (seg || (pass && nseg > 1)) load(seg);
        chunks(seg, [&](int c, uint32_t key) {
          const bool zero = key == kZero;
          zeros += __popcll(__ballot(zero));
          if ((((key ^ prefix) & hmask) | (zero ? 1u : 0u)) == 0u) atomicAdd(&sh.hist[(key >> shift) & (nb - 1)], 1);
        });
      }
      if (((kZero ^ prefix) & hmask) == 0 && lane == 0 && zeros) atomicAdd(&sh.hist[(kZero >> shift) & (nb - 1)], zeros);
      lds_sync();
      int bin, above, count;
      hist_pick<kSelThreads>(sh, nb, need, bin, above, count);
      prefix |= static_cast<uint32_t>(bin) << shift;
      need -= above;
    }
    T = prefix;
  }
  int eq_base = 0, mov_base = 0, gap_base = 0;  // of the segments before
  // The masks and ranks of a segment's chunks
  auto masks = [&](int seg) {
    chunks(seg, [&](int c, uint32_t key) {
      const unsigned long long g = __ballot(key > T), e = __ballot(key == T);
      if (lane == 0 && c < CH) sh.a[c] = g, sh.b[c] = e;
    });
    lds_sync();
    const int p0 = (seg * CH + tid) * kWave;
    const bool mine = tid < CH && p0 < nc;
    const unsigned long long gt = mine ? sh.a[tid] : 0ull, eq = mine ? sh.b[tid] : 0ull;
    auto scan = [&](int v, int which, int& all) {  // v of the threads before, and of all
      const int incl = wave_incl_scan(v, lane);
      if (lane == kWave - 1) sh.sums[which][wave] = incl;
      lds_sync();
      int before = incl - v;
      all = 0;
#pragma unroll
      for (int i = 0; i < kSelWaves; ++i) {
        const int s = sh.sums[which][i];
        before += i < wave ? s : 0;
        all += s;
      }
      return before;
    };
    int all;
    const int ne = __popcll(eq), before = eq_base + scan(ne, 0, all);
    eq_base += all;
    const unsigned long long large = gt | low_bits(eq, min(max(need - before, 0), ne)), low = bits_below(H, p0);
    const unsigned long long mov = large & ~low, gap = mine ? ~large & low : 0ull;
    const int mov_at = mov_base + scan(__popcll(mov), 1, all);
    mov_base += all;
    const int gap_at = gap_base + scan(__popcll(gap), 2, all);
    gap_base += all;
    if (mine) sh.a[tid] = mov, sh.b[tid] = gap, sh.a0[tid] = mov_at, sh.b0[tid] = gap_at;
    lds_sync();
  };
  const unsigned long long below = lanes_below(lane);
  for (int seg = 0; seg < nseg; ++seg) {
    if (nseg > 1) {
      __syncthreads();  // (the segment before has been read)
      load(seg);
      lds_sync();
    }
    masks(seg);
    const int nch = (min(SEG, nc - seg * SEG) + kWave - 1) / kWave, c0 = max(H - seg * SEG, 0) / kWave;  // (none wholly below H)
    for (int c = c0 + wave; c < nch; c += kSelWaves) {
      const unsigned long long m = sh.a[c];
      const int at = sh.a0[c] + __popcll(m & below);
      if ((m >> lane) & 1) (nseg > 1 ? reinterpret_cast<uint32_t*>(movers) : sh.key)[at] = seg * SEG + c * kWave + lane;
    }
  }
  __syncthreads();
  // Places below H.  Positions read there are at or past H or stay, so in place nothing is
  // overwritten before it is read
  eq_base = mov_base = gap_base = 0;
  for (int seg = 0; seg * SEG < H; ++seg) {
    if (nseg > 1) {
      __syncthreads();
      load(seg);
      lds_sync();
      masks(seg);
    }
    const int nch = (min(SEG, H - seg * SEG) + kWave - 1) / kWave;
    for (int c0 = wave; c0 < nch; c0 += U * kSelWaves) {
      int from[U];
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = min(c0 + u * kSelWaves, nch - 1);
        const unsigned long long g = sh.b[c];
        from[u] = seg * SEG + c * kWave + lane;
        if ((g >> lane) & 1) {
          const int at = sh.b0[c] + __popcll(g & below);
          from[u] = nseg > 1 ? movers[at] : static_cast<int>(sh.key[at]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = w[min(from[u], nc - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * kSelWaves, pos = seg * SEG + c * kWave + lane;
        if (c < nch && pos < H) {
          kept[pos] = from[u];
          if (!p.in_place || from[u] != pos) wo[pos] = v[u];
        }
      }
    }
  }
  // the last `recent`; in place through the workspace, for they may overlap their places
  float* held = p.held_w + row;
  for (int j = tid; j < p.recent; j += kSelThreads) {
    kept[H + j] = nc + j;
    (p.in_place ? held : wo + H)[j] = w[nc + j];
  }
  if (p.in_place) {
    __threadfence_block();
    __syncthreads();
    for (int j = tid; j < p.recent; j += kSelThreads) wo[H + j] = held[j];
  }
  for (int j = p.keep + tid; j < wlen; j += kSelThreads) wo[j] = 0.f;
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
  if (p.Lmax <= 4096) hipLaunchKernelGGL(evict_select_kernel<4096>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(evict_select_kernel<32768>, grid, block, 0, st, p);
  if (p.fp8) launch_evict_moves<true>(p, st);
  else launch_evict_moves<false>(p, st);
  return hipGetLastError();
}

}  // namespace saga
