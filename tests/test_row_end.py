"""The last pieces of a matrix's rows (jitnn_amd/csrc/row_end.h), driven on the CPU: no load leaves the matrix, whatever its size."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_row_end(tmp_path):
    exe = tmp_path / "row_end_test"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", str(ROOT / "jitnn_amd" / "csrc"),
                    str(ROOT / "tests" / "row_end_test.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
