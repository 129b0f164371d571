"""The serving operators at the ends of their ranges, without a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("flags", [("-O2",), ("-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined")], ids=["plain", "checked"])
def test_lines_of_steps_of_long_sequences(flags, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "check")
    subprocess.run(["g++", *flags, "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "csrc", "long_lines_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr
