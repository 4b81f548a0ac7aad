"""The scope that makes a context's device the current one (csrc/internal.hpp), on the host with a runtime of three devices
in which device 2 cannot be asked for."""
import subprocess
from pathlib import Path

import pytest

SRC = Path(__file__).resolve().parent.parent / "test-burn_b200" / "csrc"

PROGRAM = r"""
#include "internal.hpp"
#include <cstdio>
static int current = 0, sets = 0;
static bool answers = true;
extern "C" cudaError_t cudaGetDevice(int *d) { if (!answers) return cudaErrorInvalidDevice; *d = current; return cudaSuccess; }
extern "C" cudaError_t cudaSetDevice(int d) { ++sets; if (d < 0 || d > 2) return cudaErrorInvalidDevice; current = d; return cudaSuccess; }
int main()
{
    for (int before = 0; before < 3; ++before)
        for (int wanted = 0; wanted < 3; ++wanted) {
            current = before;
            sets = 0;
            {
                mf::DeviceScope scope(wanted);
                if (current != wanted) return 1;
                {
                    mf::DeviceScope inner((wanted + 1) % 3);
                    if (current != (wanted + 1) % 3) return 2;
                }
                if (current != wanted) return 3;
            }
            if (current != before) return 4;
            if (before == wanted && sets != 2) return 5;  // nothing but the inner scope's two
        }
    answers = false;
    current = 1;
    { mf::DeviceScope scope(0); if (current != 0) return 6; }
    return 0;
}
"""


def test_device_scope(tmp_path):
    cuda = Path("/usr/local/cuda/include")
    if not cuda.exists():
        pytest.skip("no CUDA headers")
    (tmp_path / "scope.cpp").write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-O1", f"-I{SRC}", f"-I{cuda}", str(tmp_path / "scope.cpp"), "-o", str(tmp_path / "scope")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "scope")], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
