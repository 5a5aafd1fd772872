"""Which tiles the GPU tests' sizes take (CPU: the rules are host code)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_half_plan_cases(tmp_path):
    exe = tmp_path / "half_plan_cases"
    build = subprocess.run(["g++", "-O2", "-std=c++20", f"-I{ROOT / 'rushlite_amd' / 'csrc' / 'hip'}",
                            str(ROOT / "tests" / "native" / "half_plan_cases.cpp"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "half plan cases ok" in out.stdout, out.stdout + out.stderr
