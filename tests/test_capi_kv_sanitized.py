"""The host code of appends with norms, 8-bit caches, attention weights and
evictions under AddressSanitizer and UndefinedBehaviorSanitizer: capi.hip,
sanitized on its host side, linked with a fuzzer (tests/sanitize/capi_kv_fuzz.cpp)
of valid and spoiled descriptors.  CPU only, as tests/test_capi_sanitized.py."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"
CLANG = "/opt/rocm/bin/amdclang++"
SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
       "-Xarch_host", "-fno-sanitize-recover=all", "-Xarch_host", "-fno-omit-frame-pointer"]


@pytest.mark.skipif(not (os.path.exists(HIPCC) and os.path.exists(CLANG)), reason="ROCm compilers not found")
@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="fuzzes with fake device pointers: hosts without a GPU only")
def test_kv_entry_points_under_asan_and_ubsan(tmp_path):
    lib = os.path.join(ROOT, "saga_amd", "libsaga_amd.so")
    if not os.path.exists(lib):
        pytest.skip("libsaga_amd.so not built")
    common = ["--offload-arch=gfx950", "-O1", "-g", "-std=c++17", "-fPIC",
              "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-I", os.path.join(ROOT, "include")]
    capi_o, fuzz_o, exe = (str(tmp_path / n) for n in ("capi_asan.o", "fuzz.o", "capi_kv_fuzz"))
    for src, obj in ((os.path.join(ROOT, "saga_amd", "csrc", "capi.hip"), capi_o),
                     (os.path.join(ROOT, "tests", "sanitize", "capi_kv_fuzz.cpp"), fuzz_o)):
        r = subprocess.run([HIPCC, *common, *SAN, "-c", src, "-o", obj], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([CLANG, "-fsanitize=address,undefined", fuzz_o, capi_o, lib, "-L/opt/rocm/lib", "-lamdhip64",
                        f"-Wl,-rpath,{os.path.dirname(lib)}", "-Wl,-rpath,/opt/rocm/lib", "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe, "300000"], capture_output=True, text=True, env=env, timeout=300)
    print(r.stdout[-500:])
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-4000:])
    assert "rejected" in r.stdout and "Sanitizer" not in r.stderr, r.stderr[-4000:]
