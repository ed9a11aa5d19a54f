"""Launch arithmetic of the microscaled linear layer on the host, from the
header that its kernels and launchers use, with the compiler's check of signed
overflow, which ends the program."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "test-model-thing-cuda_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None,
                                reason="hipcc not available")


def _run(tmp_path, program):
    src, exe = tmp_path / "launch.hip", tmp_path / "launch"
    src.write_text(program)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-I", CSRC,
                        "-Xarch_host", "-fsanitize=signed-integer-overflow",
                        "-Xarch_host", "-fsanitize-trap=signed-integer-overflow",
                        str(src), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout)


WIDEST = r"""
#include <cstdio>
#include "linear.hpp"
int main() {
    const int widths[] = {32, 64, 96, 128, 224, 256, 288, 4096, 1 << 22, 2147483392, 2147483424, 2147483616};
    for (int K : widths) {
        const int64_t cols = K >= 256 ? 256 : K >= 128 ? 128 : 64, tiles = ((int64_t)K + cols - 1) / cols;
        if (tmt::mx_tiles_per_row(K) != tiles || tmt::mx_tiles(1, K) != tiles) {
            std::printf("K %d: %d tiles a row\n", K, tmt::mx_tiles_per_row(K));
            return 1;
        }
    }
    std::printf("ok\n");
    return 0;
}
"""


def test_tiles_of_the_widest_rows(tmp_path):
    """Rows of any multiple of 32 columns that 32 bits hold."""
    _run(tmp_path, WIDEST)
