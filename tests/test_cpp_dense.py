"""The dense path through the C++ host layer (include/mako_h3.hpp): tests/cpp/h3_dense_test, built by
__graft_entry__.build(), runs every member on the GPU and checks it against double on the host."""
import subprocess
from pathlib import Path

import pytest

EXE = Path(__file__).resolve().parent / "cpp" / "h3_dense_test"


def test_driver_is_built_and_links():
    assert EXE.exists(), "run __graft_entry__.build()"
    out = subprocess.run(["ldd", str(EXE)], capture_output=True, text=True, check=True).stdout
    assert "not found" not in out, out
    assert "libmako_h3.so" in out


@pytest.mark.gpu
def test_host_layer(dev):
    r = subprocess.run([str(EXE)], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "FAIL" not in r.stdout
