"""A GPU run that ends at its first failure runs everything before the test that needs the reference's sources."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_the_tensor_library_does_not_hide_other_tests():
    r = subprocess.run([sys.executable, "-m", "pytest", "tests", "-m", "gpu", "--collect-only", "-q"], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    tests = [line for line in r.stdout.splitlines() if "::" in line]
    here = [i for i, t in enumerate(tests) if "test_gpu_bee_tensor.py" in t]
    assert len(tests) > 1000 and len(here) == 1, r.stdout[-2000:] + r.stderr
    if not (ROOT / "oracle" / "_ref" / "test_bee_tensor_cuda").exists():
        assert here[0] == len(tests) - 1
