"""The host bookkeeping of 8-bit blocks and eviction under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only): test_host_asan.py's build of kvc_host.cpp,
rerunning test_q8_bookkeeping.py and test_evict_index.py (host-only contexts)."""
import os
import subprocess
import sys

import pytest

from test_host_asan import HIPCC, PKG, ROOT, _asan_runtime


def test_8_bit_and_eviction_bookkeeping_clean_under_sanitizers(tmp_path):
    rt = _asan_runtime()
    kobj = PKG / "_build" / "kvc_kernels.o"
    if rt is None or not HIPCC.exists():
        pytest.skip("no hipcc / clang ASan runtime in this image")
    if not kobj.exists():
        pytest.skip("kernel object not built (run __graft_entry__.build())")
    if os.environ.get("LD_PRELOAD"):
        pytest.skip("a preload is already set in this environment; it is not replaced")
    hobj, lib = tmp_path / "kvc_host_asan.o", tmp_path / "libkvc.so"
    host = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined"]
    subprocess.run([str(HIPCC), "-O1", "-g", "-std=c++17", "-fPIC", "-x", "hip", "--offload-arch=gfx950", *host,
                    "-Xarch_host", "-fno-sanitize-recover=undefined", "-fno-omit-frame-pointer", f"-I{PKG / 'csrc'}",
                    f"-I{ROOT / 'include'}", "-c", str(PKG / "csrc" / "kvc_host.cpp"), "-o", str(hobj)],
                   check=True, capture_output=True)
    subprocess.run([str(HIPCC), "-shared", "--offload-arch=gfx950", *host, "-o", str(lib), str(kobj), str(hobj),
                    "-Wl,-rpath,/opt/rocm/lib"], check=True, capture_output=True)
    env = dict(os.environ, KVC_LIB_PATH=str(lib), LD_PRELOAD=rt,
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "not gpu", "-p", "no:cacheprovider",
                        str(ROOT / "tests" / "test_q8_bookkeeping.py"), str(ROOT / "tests" / "test_evict_index.py")],
                       cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout[-4000:], r.stderr[-4000:])
    assert " passed" in r.stdout
    assert "AddressSanitizer" not in r.stderr and "runtime error" not in r.stderr
