"""A buffer that a larger one replaces (jitnn_amd/csrc/scratch.h), driven on the CPU: what a model's experts have is not lost where there is no room for more."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_replace_buffer(tmp_path):
    exe = tmp_path / "replace_buffer_test"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", str(ROOT / "jitnn_amd" / "csrc"),
                    str(ROOT / "tests" / "replace_buffer_test.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
