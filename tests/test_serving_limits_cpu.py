"""The serving operators at the ends of their ranges, without a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHECKED = ("-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined")


def _run_check(name, flags, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "check")
    subprocess.run(["g++", *flags, "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "csrc", name)], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


@pytest.mark.parametrize("flags", [("-O2",), CHECKED], ids=["plain", "checked"])
def test_lines_of_steps_of_long_sequences(flags, tmp_path):
    _run_check("long_lines_check.cpp", flags, tmp_path)


def test_steps_outside_a_line_belong_to_its_ends(tmp_path):
    """Offsets of packed sequences that overlap: what a kernel reads for a step that is not on its line has to exist."""
    _run_check("shares_check.cpp", CHECKED, tmp_path)
