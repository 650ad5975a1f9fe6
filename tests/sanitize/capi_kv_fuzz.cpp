// Random and near-valid descriptors through the entry points of appends with
// norms, 8-bit caches, attention weights and evictions, with AddressSanitizer and
// UndefinedBehaviorSanitizer on the host code of capi.hip.  Every call must return
// (an error, or past validation a launch that fails for want of a device) without
// a sanitizer report, and every entry point must be reached past its checks; this
// program refuses to run where a GPU is visible.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include "saga_amd.h"

namespace {

uint64_t g_state = 0x2545f4914f6cdd1dull;

uint64_t next() {  // xorshift*
  g_state ^= g_state >> 12;
  g_state ^= g_state << 25;
  g_state ^= g_state >> 27;
  return g_state * 0x9e3779b97f4a7c15ull;
}

template <class T, size_t N>
T pick(const T (&a)[N]) {
  return a[next() % N];
}

const int64_t kOdd[] = {-1, 0, 1, 2, 3, 15, 16, 31, 33, 64, 127, 1024, int64_t(1) << 25, int64_t(1) << 31, int64_t(1) << 40,
                        INT64_MAX, INT64_MIN};

saga_tensor contig(int32_t dtype, std::initializer_list<int64_t> shape) {
  saga_tensor t;
  std::memset(&t, 0, sizeof t);
  t.data = reinterpret_cast<void*>(uintptr_t{0x100000});
  t.dtype = dtype;
  t.ndim = static_cast<int32_t>(shape.size());
  int i = 0;
  for (int64_t n : shape) t.shape[i++] = n;
  uint64_t acc = 1;
  for (i = t.ndim - 1; i >= 0; --i) {
    t.stride[i] = static_cast<int64_t>(acc);
    acc *= static_cast<uint64_t>(t.shape[i]);
  }
  return t;
}

// Leaves a descriptor as it is most of the time, else breaks one of its fields.
saga_tensor spoil(saga_tensor t) {
  switch (next() % 24) {
    case 0: t.data = reinterpret_cast<void*>(uintptr_t{next() % 2 ? 0u : 0x100002u}); break;
    case 1: t.dtype = static_cast<int32_t>(next() % 9) - 1; break;
    case 2: t.ndim = static_cast<int32_t>(next() % 7) - 1; break;
    case 3: t.shape[next() % 4] = pick(kOdd); break;
    case 4: t.stride[next() % 4] = pick(kOdd); break;
    default: break;
  }
  return t;
}

const int64_t kSmall[] = {1, 2, 3, 5, 12, 16};

saga_kv_fp8 cache(int64_t B, int64_t n_k, int64_t n_v, int64_t L, int64_t d, int64_t block) {
  const int64_t blocks = L > 0 && block > 0 ? (L - 1) / block + 1 : L;
  saga_kv_fp8 c;
  c.k_codes = spoil(contig(SAGA_DTYPE_U8, {B, n_k, L, d}));
  c.k_scales = spoil(contig(SAGA_DTYPE_F32, {B, n_k, blocks}));
  c.v_codes = spoil(contig(SAGA_DTYPE_U8, {B, n_v, L, d}));
  c.v_scales = spoil(contig(SAGA_DTYPE_F32, {B, n_v, blocks}));
  c.block = next() % 32 ? block : pick(kOdd);
  return c;
}

int64_t divisor(int64_t a, int64_t b) {
  int64_t g = 1;
  for (int64_t i = 2; i <= a; ++i)
    if (a % i == 0 && b % i == 0 && next() % 2) g = i;
  return next() % 16 ? g : pick(kSmall);
}

}  // namespace

int main(int argc, char** argv) {
  int devices = 0;
  if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
    std::fprintf(stderr, "a GPU is visible: not run\n");
    return 2;
  }
  const long calls = argc > 1 ? std::atol(argv[1]) : 100000;
  int32_t* idx = reinterpret_cast<int32_t*>(uintptr_t{0x300000});
  const float* table = reinterpret_cast<const float*>(idx);
  void* ws = reinterpret_cast<void*>(uintptr_t{0x400000});
  long rejected = 0, launched = 0, reached[7] = {};
  for (long i = 0; i < calls; ++i) {
    const int64_t n_k = pick(kSmall), n_v = pick(kSmall), B = pick(kSmall), n_q = n_k * n_v;
    const int64_t blocks[] = {32, 64, 128};
    const int64_t d = next() % 2 ? 128 : 64, block = pick(blocks);
    const int64_t L = next() % 16 ? 1 + static_cast<int64_t>(next() % 5000) : pick(kOdd);
    const int32_t dts[] = {SAGA_DTYPE_BF16, SAGA_DTYPE_F16, SAGA_DTYPE_F32};
    const int32_t dt = pick(dts);
    const saga_kv_fp8 c = cache(B, n_k, n_v, L, d, block);
    const saga_kv_fp8* cp = next() % 32 ? &c : nullptr;
    const int64_t N = next() % 16 ? B : pick(kOdd), Lw = L > 0 && L < 100000 ? L + static_cast<int64_t>(next() % 3) : 7;
    const size_t ws_bytes = next() % 8 ? size_t{1} << 40 : 64;
    void* w = next() % 8 ? ws : nullptr;
    const int which = static_cast<int>(next() % 8);
    int rc = 0;
    switch (which) {
      case 0: case 1: {
        saga_tensor x = spoil(contig(dt, {N, (n_q + n_k + n_v) * d})), o = spoil(contig(dt, {N, n_q, d}));
        saga_tensor qn = spoil(contig(dt, {d})), kn = spoil(contig(dt, {d}));
        const saga_tensor *qp = next() % 2 ? &qn : nullptr, *kp = next() % 2 ? &kn : nullptr;
        const int64_t heads = next() % 16 ? n_q : pick(kOdd);
        const float* t = next() % 8 ? table : nullptr;
        const int32_t* at = next() % 8 ? idx : nullptr;
        if (which == 0) {
          saga_tensor k = spoil(contig(dt, {B, n_k, L, d})), v = spoil(contig(dt, {B, n_v, L, d}));
          rc = saga_norm_rope_kv_append(&x, heads, t, qp, kp, 1e-6f, at, next() % 2 ? idx : nullptr, &o, &k, &v, nullptr);
        } else {
          rc = saga_norm_rope_kv_append_fp8(&x, heads, t, qp, kp, 1e-6f, at, next() % 2 ? idx : nullptr,
                                            next() % 8 ? B : pick(kOdd), &o, cp, nullptr);
        }
        break;
      }
      case 2: {
        saga_tensor k = spoil(contig(dt, {N, n_k, d})), v = spoil(contig(dt, {N, n_v, d}));
        rc = saga_kv_fp8_read(cp, next() % 8 ? idx : nullptr, next() % 2 ? idx : nullptr, &k, &v, nullptr);
        break;
      }
      case 3: case 4: {
        saga_tensor q = spoil(contig(dt, {B, n_q, 1, d})), o = spoil(contig(dt, {B, n_q, 1, d}));
        saga_tensor m = spoil(contig(next() % 2 ? SAGA_DTYPE_BOOL : dt, {B, next() % 2 ? n_q : 1, 1, Lw}));
        const saga_tensor* mp = next() % 2 ? &m : nullptr;
        const int32_t* len = next() % 2 ? idx : nullptr;
        if (which == 3) {
          saga_tensor wt = spoil(contig(SAGA_DTYPE_F32, {B, divisor(n_k, n_v), Lw}));
          rc = saga_dense_decode_fp8(&q, cp, mp, len, 0.125f, &o, next() % 2 ? &wt : nullptr, static_cast<int32_t>(next() % 2),
                                     w, ws_bytes, nullptr);
        } else {
          saga_tensor k = spoil(contig(dt, {B, n_k, L, d})), wt = spoil(contig(SAGA_DTYPE_F32, {B, divisor(n_k, n_k), Lw}));
          rc = saga_attention_weights(&q, &k, mp, len, 0.125f, &wt, static_cast<int32_t>(next() % 2), w, ws_bytes, nullptr);
        }
        break;
      }
      case 5: case 6: {
        const int64_t G = divisor(n_k, n_v), keep = next() % 16 ? 1 + static_cast<int64_t>(next() % 5000) : pick(kOdd);
        const int64_t recent = next() % 8 && keep > 0 ? static_cast<int64_t>(next() % static_cast<uint64_t>(keep)) : pick(kOdd);
        const int64_t Lo = keep > 0 && keep < 100000 ? keep + static_cast<int64_t>(next() % 3) : 5;
        saga_tensor wt = spoil(contig(SAGA_DTYPE_F32, {B, G, Lw})), wo = spoil(contig(SAGA_DTYPE_F32, {B, G, Lo}));
        const bool out = next() % 2, odd = next() % 16 == 0;
        const auto away = [](saga_tensor& t) {  // results lie elsewhere, mostly
          if (t.data && next() % 16) t.data = reinterpret_cast<void*>(reinterpret_cast<uintptr_t>(t.data) + (1u << 24));
        };
        away(wo);
        const int32_t* len = next() % 8 ? idx : nullptr;
        int32_t* kept = next() % 8 ? idx : nullptr;
        if (which == 5) {
          saga_tensor k = spoil(contig(dt, {B, n_k, L, d})), v = spoil(contig(dt, {B, n_v, L, d}));
          saga_tensor ko = spoil(contig(dt, {B, n_k, Lo, d})), vo = spoil(contig(dt, {B, n_v, Lo, d}));
          away(ko), away(vo);
          rc = saga_evict_kv(&k, &v, &wt, len, keep, recent, out ? &ko : nullptr, out != odd ? &vo : nullptr,
                             out ? &wo : nullptr, kept, w, ws_bytes, nullptr);
        } else {
          saga_kv_fp8 co = cache(B, n_k, n_v, Lo, d, block);
          for (saga_tensor* t : {&co.k_codes, &co.k_scales, &co.v_codes, &co.v_scales}) away(*t);
          rc = saga_evict_kv_fp8(cp, &wt, len, keep, recent, out ? &co : nullptr, out != odd ? &wo : nullptr, kept, w, ws_bytes,
                                 nullptr);
        }
        break;
      }
      default:
        saga_dense_fp8_workspace_bytes(pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd), static_cast<int32_t>(next() % 2));
        saga_attention_weights_workspace_bytes(pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd));
        saga_evict_workspace_bytes(pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd),
                                   static_cast<int32_t>(next() % 2));
        continue;
    }
    if (rc == SAGA_ERR_HIP) ++launched, ++reached[which];
    else if (rc < 0) ++rejected;
  }
  std::printf("%ld calls: %ld rejected, %ld reached the launch (%ld %ld %ld %ld %ld %ld %ld)\n", calls, rejected, launched,
              reached[0], reached[1], reached[2], reached[3], reached[4], reached[5], reached[6]);
  for (long n : reached)
    if (!n) return 1;
  return rejected > 0 ? 0 : 1;
}
