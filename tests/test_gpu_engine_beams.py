"""Runs the C++ beam search tests (tests/cpp/test_beams.cpp) on the GPU:
kvengine::generate_beams over fork, shared decode, selection and reorder.  The
binary is built by __graft_entry__.build() (make -C tests/cpp)."""
import subprocess
from pathlib import Path

import pytest

BIN = Path(__file__).resolve().parent / "cpp" / "test_beams"


@pytest.mark.gpu
def test_cpp_beam_search():
    if not BIN.exists():
        pytest.fail(f"{BIN} is not built (make -C tests/cpp)")
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, f"test_beams exited {r.returncode}:\n{r.stdout}\n{r.stderr}"
    assert "check failed" not in r.stderr
