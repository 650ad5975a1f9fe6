// What keeps a cache short: the softmax weight that every cached position gathers over a step's
// query heads, and the eviction of the positions that gathered least.
#include <algorithm>

#include "fp8.cuh"
#include "kernels.h"
#include "select.cuh"
#include "weights.cuh"

namespace saga {

// ---- weights per position (weights.cuh) ----

__global__ void __launch_bounds__(256) attention_weights_kernel(WeightsParams p) { attention_weights(p, blockIdx.x); }

hipError_t launch_attention_weights(const WeightsParams& p, hipStream_t st) {
  const int64_t blocks = attention_weights_blocks(p);
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
  alignas(16) uint32_t key[SEG];  // ranking keys, four positions' together, of each 32 positions in an order of their own
  int hist[2048];
  int cnt[kSelWaves];
  int sel_bin, sel_above, sel_cnt;
  int sums[4][kSelWaves];
};

// A weight as what it is ranked by: any NaN above all numbers, -0 as 0; never 0, which stands for no position.
__device__ __forceinline__ uint32_t rank_key(float w) { return f32_to_key(w == w ? w + 0.f : __uint_as_float(0x7fffffffu)); }

// The lowest `count` set bits of m.
__device__ __forceinline__ uint32_t low_bits(uint32_t m, int count) {
  if (count == 0) return 0u;
  const int drop = __popc(m) - count;
  for (int i = 0; i < drop; ++i) m &= ~(1u << (31 - __clz(static_cast<int>(m))));
  return m;
}

// Bits of positions below `end` of 32 that start at p0.
__device__ __forceinline__ uint32_t bits_below(int end, int p0) {
  const int n = min(max(end - p0, 0), 32);
  return n == 0 ? 0u : ~0u >> (32 - n);
}

// One block per (batch row, group), a segment of SEG positions' ranking keys in LDS (a row of one
// segment is read once, longer ones for every pass).  The H-th largest key by radix (11, 11, 10
// bits), equal ones by position: the first digits are counted as the row is read; the other two, of a
// row of one segment, over the keys that share the H-th's.  What is large of 32 positions is one
// mask, a thread's: every prefix of the selection is one scan of the block.  The result is, per 32
// places below H, the mask of their gaps and the first one's rank, and the positions that move there
// in order; what to do with them is the moving blocks' work, of which there are many.
// One CU's work: 8 x 32769 positions 18.5 us, of which the row's 128 KB take 5 (what one CU gets from
// memory; 16 or 32 loads in flight for 8, or 16 bytes each, no less), 20 rows of 8195 15.5; rows of several
// segments, read four times, 57 (8 x 65541) and 107 (4 x 131072).  Measured before: 82 us with keys in
// registers and code unrolled over them, 22 with masks by ballots over 64 positions a wave.
template <int SEG>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
  __shared__ SelShared<SEG> sh;
  static_assert(SEG <= 32 * kSelThreads && SEG % (4 * kSelThreads) == 0, "32 positions a thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bi = blockIdx.x / p.G, gi = blockIdx.x - bi * p.G;
  const int n = min(max(p.kv_len[bi], 0), p.Lmax);
  if (n <= p.keep) return;
  const float* w = p.w + bi * p.w_sb + gi * p.w_sg;
  const int64_t row = blockIdx.x;
  const int H = p.keep - p.recent, nc = n - p.recent;  // candidates: [0, nc), nc > H
  const int nseg = (nc + SEG - 1) / SEG;
  constexpr uint32_t kZero = 0x80000000u;
  // f(key) of this thread's positions of a segment as they are read into LDS, 0 behind nc to the end of
  // a round.  Units of four positions are permuted within their 32, so that threads that each read
  // their 32 meet other banks.
  constexpr int U = SEG < 8 * kSelThreads ? SEG / kSelThreads : 8, ROUND = U * kSelThreads;
  const int own = (tid & ~31) | ((((tid >> 2) ^ (tid >> 5)) & 7) << 2) | (tid & 3);
  auto load = [&](int seg, auto f) {
    const int end = nc - seg * SEG, whole = min(SEG, end);
    float next[U];
    auto fetch = [&](int j0) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = w[seg * SEG + min(j0 + u * kSelThreads + tid, end - 1)];
    };
    fetch(0);
    for (int j0 = 0; j0 < whole; j0 += ROUND) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = next[u];
      if (j0 + ROUND < whole) fetch(j0 + ROUND);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t key = j0 + u * kSelThreads + tid < end ? rank_key(v[u]) : 0u;
        sh.key[j0 + u * kSelThreads + own] = key;
        f(key);
      }
    }
  };
  // f(key) of the segment's positions, a wave's those that it has read (other lanes of it wrote them:
  // between wave_syncs)
  auto each = [&](int seg, auto f) {
    for (int j0 = 0; j0 < min(SEG, nc - seg * SEG); j0 += 4 * kSelThreads) {
      uint32_t key[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) key[u] = sh.key[j0 + u * kSelThreads + tid];
#pragma unroll
      for (int u = 0; u < 4; ++u) f(key[u]);
    }
  };
  auto key_of = [&](int i) { return sh.key[tid * 32 + ((((i >> 2) ^ tid) & 7) << 2) + (i & 3)]; };
  // The masks of keys above `top` and of keys in [from, top] of this thread's positions of a segment
  uint32_t gt = 0, eq = 0;
  auto masks = [&](int seg, uint32_t from, uint32_t top) {
    gt = eq = 0;
    if (tid * 32 >= min(SEG, nc - seg * SEG)) return;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(&sh.key[tid * 32 + (((i ^ tid) & 7) << 2)]);
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        gt = 2 * gt + (k[e] > top ? 1u : 0u);
        eq = 2 * eq + (k[e] >= from ? 1u : 0u);
      }
    }
    eq &= ~gt;
  };
  auto wave_part = [&](int v, int which) {  // v of the wave's threads before
    const int incl = wave_incl_scan(v, lane);
    if (lane == kWave - 1) sh.sums[which][wave] = incl;
    return incl - v;
  };
  auto block_part = [&](int which, int& all) {  // of the waves before, and of all
    int before = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
      const int s = sh.sums[which][i];
      before += i < wave ? s : 0;
      all += s;
    }
    return before;
  };

  uint32_t T = 0xffffffffu;  // the H-th largest key
  int need = 0;              // of those equal to it, the first `need` stay
  bool held = false;         // gt and eq hold the row's masks already
  for (int i = tid; i < 2048; i += kSelThreads) sh.hist[i] = 0;
  lds_sync();
  {
    int zeros = 0;  // weights of 0 may be many: counted by the wave
    for (int seg = 0; seg < nseg; ++seg) {
      load(seg, [&](uint32_t key) {
        zeros += __popcll(__ballot(key == kZero));
        if (key << 1) atomicAdd(&sh.hist[key >> 21], 1);
      });
    }
    if (zeros && lane == 0) atomicAdd(&sh.hist[kZero >> 21], zeros);
  }
  lds_sync();
  if (H > 0) {
    need = H;
    int bin, above, count;
    hist_pick<kSelThreads>(sh, 2048, need, bin, above, count);
    uint32_t prefix = static_cast<uint32_t>(bin) << 21;
    need -= above;
    held = nseg == 1;
    if (held) masks(0, prefix, prefix | 0x1fffffu);
#pragma unroll 1
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = pass == 1 ? 10 : 0, nb = pass == 1 ? 2048 : 1024;
      const uint32_t hmask = pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < 2048; i += kSelThreads) sh.hist[i] = 0;
      lds_sync();
      int zeros = 0;
      auto count_key = [&](uint32_t key) {
        const bool zero = key == kZero;
        zeros += zero ? 1 : 0;
        if ((((key ^ prefix) & hmask) | (zero ? 1u : 0u)) == 0u) atomicAdd(&sh.hist[(key >> shift) & (nb - 1)], 1);
      };
      if (held) {
        for (uint32_t m = eq; m; m &= m - 1) count_key(key_of(__builtin_ctz(m)));
      } else {
        for (int seg = 0; seg < nseg; ++seg) {
          load(seg, [](uint32_t) {});
          wave_sync();
          each(seg, count_key);
          wave_sync();  // (the next segment's keys overwrite them)
        }
      }
      if (((kZero ^ prefix) & hmask) == 0) {
        zeros = wave_incl_scan(zeros, lane);
        if (lane == kWave - 1 && zeros) atomicAdd(&sh.hist[(kZero >> shift) & (nb - 1)], zeros);
      }
      lds_sync();
      hist_pick<kSelThreads>(sh, nb, need, bin, above, count);
      prefix |= static_cast<uint32_t>(bin) << shift;
      need -= above;
    }
    T = prefix;
    if (held) {  // of the H-th's bin: above T, and T
      uint32_t same = 0;
      for (uint32_t m = eq; m; m &= m - 1) {
        const uint32_t key = key_of(__builtin_ctz(m));
        if (key > T) gt |= m & -m;
        if (key == T) same |= m & -m;
      }
      eq = same;
    }
  }
  const int nplace = (p.keep + 31) / 32;
  int32_t* movers = p.movers + row * p.keep;
  int eq_base = 0, moved = 0, opened = 0;  // of the segments before
  for (int seg = 0; seg < nseg; ++seg) {
    if (nseg > 1) {
      __syncthreads();  // (the segment before has been read)
      load(seg, [](uint32_t) {});
      lds_sync();
    }
    if (!held) masks(seg, T, T);
    const int p0 = seg * SEG + tid * 32, ne = __popc(eq), eq_at = wave_part(ne, 1);
    lds_sync();
    int all;
    const int before = eq_base + eq_at + block_part(1, all);
    eq_base += all;
    const uint32_t large = gt | low_bits(eq, min(max(need - before, 0), ne)), low = bits_below(H, p0);
    const uint32_t mov = large & ~low, gap = tid * 32 < SEG ? ~large & low : 0u;
    const int mov_at = wave_part(__popc(mov), 2), gap_at = wave_part(__popc(gap), 3);
    lds_sync();
    int k = moved + mov_at + block_part(2, all);
    moved += all;
    for (uint32_t m = mov; m; m &= m - 1) movers[k++] = p0 + __builtin_ctz(m);
    k = opened + gap_at + block_part(3, all);
    opened += all;
    if (tid * 32 < SEG && p0 < p.keep) {
      p.gap[row * nplace + p0 / 32] = gap;
      p.gap_at[row * nplace + p0 / 32] = k;
    }
  }
}

// Rows to their places: a block of threads per (batch row, head, 128 places); the heads behind keys and
// values are the groups' weights, whose blocks write `kept` too.  FP8: a block of S places takes
// the largest of its rows' scales and a row from under a smaller one is rounded to it.  PHASE 0:
// into other tensors.  In place, two launches: 1: the places below staged0 (a multiple of S), whose
// rows come from at or above it or stay, and the rows of the end into the stage; 2: from the stage to
// the end, and zeros for the weights behind.  PIECES: 16 bytes each of a row; a thread's are all in
// flight while the scales are compared.
// Bound by the rows, read once and written once: 8 x 16384 rows of 3 heads of 256 bytes (201 MB)
// 43.9 us, 4.6 TB/s; in place, where the larger part stays, 27.8 + 5.6.
constexpr int kMoveRows = 128;

template <int PHASE, bool FP8, int PIECES>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
  constexpr int PT = kMoveRows * PIECES / 256, ROWS = 256 / PIECES;  // pieces of a thread, rows side by side
  __shared__ int from_sh[kMoveRows];
  __shared__ float scale_sh[kMoveRows], top_sh[kMoveRows], wave_top[2];
  const int tid = threadIdx.x;
  const int nblk = (p.keep + kMoveRows - 1) / kMoveRows, first = PHASE == 2 ? p.staged0 / kMoveRows : 0;
  const int blocks = nblk - first + (PHASE == 1 ? 0 : 1);  // (a last one for the weights behind)
  const int kv_heads = p.rows[0].heads + p.rows[1].heads, heads = kv_heads + p.G;
  int id = blockIdx.x;
  const int blk = id % blocks + first;
  id /= blocks;
  const int hh = id % heads, bi = id / heads;
  const bool is_v = hh >= p.rows[0].heads, is_w = hh >= kv_heads;
  const EvictRows& r = p.rows[is_v ? 1 : 0];
  const int h = is_w ? hh - kv_heads : hh - (is_v ? p.rows[0].heads : 0), gi = is_w ? h : h / (r.heads / p.G);
  const int64_t group = static_cast<int64_t>(bi) * p.G + gi;
  const int j0 = blk * kMoveRows, H = p.keep - p.recent;
  if (blk == nblk) {  // (weights only)
    float* wo = p.w_out + bi * p.wo_sb + gi * p.wo_sg;
    if (is_w)
      for (int64_t j = p.keep + tid; j < p.wo_len; j += 256) wo[j] = 0.f;
    return;
  }
  const int64_t nstage = p.keep - p.staged0;
  const int64_t srow = (static_cast<int64_t>(bi) * r.heads + h) * nstage - p.staged0;  // + place
  const int mine = j0 + tid;  // the place that this thread looks up
  int from = -1;
  float scale = 0.f;
  if (tid < kMoveRows) {
    const int64_t at = group * ((p.keep + 31) / 32) + min(mine, p.keep - 1) / 32;
    const int kv = p.kv_len[bi];
    const uint32_t gap = p.gap[at];  // (nothing is there where nothing is evicted)
    const int rank = p.gap_at[at] + __popc(gap & ((1u << (mine & 31)) - 1));
    const int n = min(max(kv, 0), p.Lmax);
    if (mine < p.keep && (PHASE != 2 || mine >= p.staged0)) {
      if (n <= p.keep) from = mine < n ? mine : -1;
      else if (mine >= H) from = n - p.keep + mine;
      else from = (gap >> (mine & 31)) & 1 ? p.movers[group * p.keep + rank] : mine;
    }
    from_sh[tid] = from;
    if (FP8 && from >= 0 && !is_w) {
      const float* ss = r.ss + bi * r.ss_sb + h * r.ss_sh;
      scale = PHASE == 2 ? r.stage_s[srow + mine] : ss[from >> p.shift];
    }
  }
  if (is_w) {
    if (tid >= kMoveRows || mine >= p.keep || (PHASE == 2 && mine < p.staged0)) return;
    float* held = p.stage_w + group * nstage - p.staged0;
    if (PHASE != 2) p.kept[group * p.keep + mine] = from;
    const float v = from < 0 ? 0.f : PHASE == 2 ? held[mine] : p.w[bi * p.w_sb + gi * p.w_sg + from];
    if (PHASE == 1 && mine >= p.staged0) held[mine] = v;
    else if (mine < p.wo_len && (PHASE != 1 || from != mine)) p.w_out[bi * p.wo_sb + gi * p.wo_sg + mine] = v;
    return;
  }
  __syncthreads();
  const char* src = r.src + bi * r.s_sb + h * r.s_sh;
  char* dst = r.dst + bi * r.d_sb + h * r.d_sh;
  float* ds = FP8 ? r.ds + bi * r.ds_sb + h * r.ds_sh : nullptr;
  const int c = tid % PIECES, row0 = tid / PIECES;
  u32x4 v[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) {  // (no branch: it would be waited for; what has no place is read from its head's first row)
    const int row = row0 + i * ROWS, at = from_sh[row];
    const char* a = PHASE == 2 ? (at < 0 ? src : r.stage + (srow + j0 + row) * PIECES * 16) : src + max(at, 0) * r.s_sl;
    v[i] = ld16(a + 16 * c);
  }
  if constexpr (FP8) {
    const int S = 1 << p.shift;
    float top = scale;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    if (S > 32) top = fmaxf(top, __shfl_xor(top, 32));
    if (tid < kMoveRows && (tid & 63) == 0) wave_top[tid >> 6] = top;
    if (tid < kMoveRows) scale_sh[tid] = scale;
    lds_sync();
    if (S > 64) top = fmaxf(wave_top[0], wave_top[1]);
    if (tid < kMoveRows) top_sh[tid] = top;
    lds_sync();
    // a block's scale, by its first row's thread, where any of its rows is there (rows of a block are there
    // from its first one on); in place it is read above by this block alone
    if (tid < kMoveRows && (mine & (S - 1)) == 0 && from >= 0 && (PHASE != 1 || mine < p.staged0)) ds[mine >> p.shift] = top;
  }
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int row = row0 + i * ROWS, at = from_sh[row], place = j0 + row;
    if (at < 0) continue;
    if (PHASE == 1 && place >= p.staged0) {
      *reinterpret_cast<u32x4*>(r.stage + ((srow + place) * PIECES + c) * 16) = v[i];
      if (FP8 && c == 0) r.stage_s[srow + place] = scale_sh[row];
      continue;
    }
    const float s = FP8 ? scale_sh[row] : 0.f, top = FP8 ? top_sh[row] : 0.f;
    if (PHASE == 1 && at == place && s == top) continue;
    if (FP8 && s != top) v[i] = fp8_rescaled(v[i], s * fp8_inverse(top));
    *reinterpret_cast<u32x4*>(dst + place * r.d_sl + 16 * c) = v[i];
  }
}

template <bool FP8, int PIECES>
static void launch_evict_moves(const EvictParams& p, hipStream_t st) {
  const int64_t nblk = (p.keep + kMoveRows - 1) / kMoveRows;
  const int64_t rows = static_cast<int64_t>(p.B) * (p.rows[0].heads + p.rows[1].heads + p.G);
  if (!p.in_place) {
    hipLaunchKernelGGL((evict_move_kernel<0, FP8, PIECES>), dim3(static_cast<unsigned>(rows * (nblk + 1))), dim3(256), 0, st, p);
    return;
  }
  hipLaunchKernelGGL((evict_move_kernel<1, FP8, PIECES>), dim3(static_cast<unsigned>(rows * nblk)), dim3(256), 0, st, p);
  const int64_t rest = nblk + 1 - p.staged0 / kMoveRows;
  hipLaunchKernelGGL((evict_move_kernel<2, FP8, PIECES>), dim3(static_cast<unsigned>(rows * rest)), dim3(256), 0, st, p);
}

hipError_t launch_evict(const EvictParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.B * p.G)), block(kSelThreads);
  if (p.Lmax <= 4096) hipLaunchKernelGGL(evict_select_kernel<4096>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(evict_select_kernel<32768>, grid, block, 0, st, p);
  const int pieces = p.rows[0].pieces;  // of a row: 64 or 128 dims of 1, 2 or 4 bytes
  if (p.fp8) {
    if (pieces == 4) launch_evict_moves<true, 4>(p, st);
    else launch_evict_moves<true, 8>(p, st);
  } else {
    if (pieces == 8) launch_evict_moves<false, 8>(p, st);
    else if (pieces == 16) launch_evict_moves<false, 16>(p, st);
    else launch_evict_moves<false, 32>(p, st);
  }
  return hipGetLastError();
}

}  // namespace saga
