"""The shared-memory limit of a kernel whose launches need different sizes, raised from two host threads at once
(tests/cpp/test_smem_limit.cpp, against a fake CUDA runtime: no GPU)."""
import subprocess
from pathlib import Path

from bee_b200 import build

ROOT = Path(__file__).resolve().parent.parent


def test_two_first_calls_at_once(tmp_path):
    exe = tmp_path / "test_smem_limit"
    subprocess.run(["g++", "-O1", "-std=c++20", "-Wall", "-I", str(ROOT / "bee_b200" / "csrc"), "-I", build.CUDA_INC,
                    str(ROOT / "tests" / "cpp" / "test_smem_limit.cpp"), "-o", str(exe), "-lpthread"], check=True)
    for _ in range(3):
        r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stdout + r.stderr
