"""The whole numbers in which the sampler holds its bins, on the CPU: a bin that holds the
largest vocabulary counts and weighs what its tokens do."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_a_bin_holds_the_largest_vocabulary(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = tmp_path / "sample_bins"
    subprocess.run(["g++", "-std=c++17", "-O2", str(HERE / "host" / "sample_bins.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
