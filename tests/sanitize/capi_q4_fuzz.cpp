// Random and near-valid descriptors through the 4-bit entry points of the C ABI,
// with AddressSanitizer and UndefinedBehaviorSanitizer on the host code of
// capi.hip.  Every call must return (an error, or past validation a launch that
// fails for want of a device) without a sanitizer report; this program refuses
// to run where a GPU is visible.
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

saga_kv_q4 cache(int64_t B, int64_t n_k, int64_t n_v, int64_t L, int64_t d, int64_t group) {
  saga_kv_q4 c;
  c.k_codes = spoil(contig(SAGA_DTYPE_U8, {B, n_k, L, d / 2}));
  c.k_scales = spoil(contig(SAGA_DTYPE_F16, {B, n_k, L, 2 * d / group}));
  c.v_codes = spoil(contig(SAGA_DTYPE_U8, {B, n_v, L, d / 2}));
  c.v_scales = spoil(contig(SAGA_DTYPE_F16, {B, n_v, L, 2 * d / group}));
  return c;
}

}  // namespace

int main(int argc, char** argv) {
  int devices = 0;
  if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
    std::fprintf(stderr, "a GPU is visible: not run\n");
    return 2;
  }
  const long calls = argc > 1 ? std::atol(argv[1]) : 100000;
  const int32_t* idx = reinterpret_cast<const int32_t*>(uintptr_t{0x300000});
  void* ws = reinterpret_cast<void*>(uintptr_t{0x400000});
  long rejected = 0, launched = 0;
  for (long i = 0; i < calls; ++i) {
    const int64_t n_k = pick(kSmall), n_v = pick(kSmall), B = pick(kSmall), n_q = n_k * n_v;
    const int64_t d = next() % 2 ? 128 : 64, group = next() % 2 ? 32 : 64;
    const int64_t L = next() % 16 ? 1 + static_cast<int64_t>(next() % 5000) : pick(kOdd);
    const int32_t dts[] = {SAGA_DTYPE_BF16, SAGA_DTYPE_F16, SAGA_DTYPE_F32};
    const int32_t dt = pick(dts);
    const saga_kv_q4 c = cache(B, n_k, n_v, L, d, group);
    const saga_kv_q4* cp = next() % 32 ? &c : nullptr;
    int rc = 0;
    switch (next() % 6) {
      case 0: {
        saga_tensor q = spoil(contig(dt, {B, n_q, 1, d})), o = spoil(contig(dt, {B, n_q, 1, d}));
        saga_tensor m = spoil(contig(next() % 2 ? SAGA_DTYPE_BOOL : dt, {B, next() % 2 ? n_q : 1, 1, L > 0 && L < 100000 ? L + 1 : 7}));
        rc = saga_dense_decode_q4(&q, cp, next() % 2 ? &m : nullptr, next() % 2 ? idx : nullptr, 0.125f, &o,
                                  next() % 8 ? ws : nullptr, next() % 8 ? size_t{1} << 40 : 64, nullptr);
        break;
      }
      case 1: {
        const int64_t N = next() % 16 ? B : pick(kOdd);
        saga_tensor x = spoil(contig(dt, {N, (n_q + n_k + n_v) * d})), o = spoil(contig(dt, {N, n_q, d}));
        rc = saga_rope_kv_append_q4(&x, next() % 16 ? n_q : pick(kOdd), next() % 8 ? reinterpret_cast<const float*>(idx) : nullptr,
                                    next() % 8 ? idx : nullptr, next() % 2 ? idx : nullptr, &o, cp, nullptr);
        break;
      }
      case 2: {
        const int64_t N = next() % 16 ? B : pick(kOdd);
        saga_tensor k = spoil(contig(dt, {N, n_k, d})), v = spoil(contig(dt, {N, n_v, d}));
        rc = saga_kv_q4_read(cp, next() % 8 ? idx : nullptr, next() % 2 ? idx : nullptr, &k, &v, nullptr);
        break;
      }
      case 3: case 4: {
        const int64_t gs[] = {32, 64, 128, 96};
        const int64_t g = pick(gs), K = g * pick(kSmall), N = 16 * pick(kSmall), M = next() % 16 ? 1 + static_cast<int64_t>(next() % 32) : pick(kOdd);
        saga_q4_weight w = {spoil(contig(SAGA_DTYPE_U8, {N / 16, (K + 127) / 128, 1024})),
                            spoil(contig(SAGA_DTYPE_F16, {N / 16, K / g, 16, 2}))};
        if (next() % 2) {
          const int32_t epi = static_cast<int32_t>(next() % 4);
          saga_tensor x = spoil(contig(SAGA_DTYPE_BF16, {M, K})), y = spoil(contig(SAGA_DTYPE_BF16, {M, epi == 2 ? N / 2 : N}));
          saga_tensor b = spoil(contig(SAGA_DTYPE_BF16, {N}));
          rc = saga_gemv_q4(&x, next() % 32 ? &w : nullptr, next() % 4 ? nullptr : &b, next() % 2 ? 1e-6f : -1.f, epi, &y,
                            next() % 2 ? ws : nullptr, size_t{1} << 30, nullptr);
        } else {
          saga_unpack_q4_item it[2];
          for (auto& e : it) e = {w, spoil(contig(SAGA_DTYPE_BF16, {N, K})), next() % 8 ? 0 : pick(kOdd), next() % 4 ? 0 : pick(kOdd)};
          rc = saga_unpack_gemv_q4(next() % 32 ? it : nullptr, next() % 16 ? 1 + static_cast<int32_t>(next() % 2) : 0, nullptr);
        }
        break;
      }
      default:
        saga_dense_q4_workspace_bytes(pick(kOdd), pick(kOdd), pick(kOdd), pick(kOdd));
        saga_gemv_q4_workspace_bytes(pick(kOdd), pick(kOdd), pick(kOdd));
        continue;
    }
    if (rc == SAGA_ERR_HIP) ++launched;
    else if (rc < 0) ++rejected;
  }
  std::printf("%ld calls: %ld rejected, %ld reached the launch\n", calls, rejected, launched);
  return rejected > 0 && launched > 0 ? 0 : 1;
}
