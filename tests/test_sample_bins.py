"""The whole numbers in which the sampler holds its bins, on the CPU: a bin that holds the
largest vocabulary counts and weighs what its tokens do."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def run(name, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = tmp_path / name
    subprocess.run(["g++", "-std=c++17", "-O2", str(HERE / "host" / (name + ".cpp")), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_a_bin_holds_the_largest_vocabulary(tmp_path):
    run("sample_bins", tmp_path)


def test_every_goal_has_a_place(tmp_path):
    """Also one that rounded masses would end in front of."""
    run("sample_places", tmp_path)
