"""The serving operators at the ends of their ranges, without a GPU."""
import os
import shutil
import subprocess

import pytest
import torch

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


def test_rows_are_aligned_or_copied():
    """Contiguous tensors at odd storage offsets are copied; strides of dimensions with one entry are no strides."""
    from flagattention_amd import serving as S

    buf = torch.zeros(4 * 64 * 10 + 8, dtype=torch.bfloat16)
    t = buf[1:-7].view(10, 4, 64)
    assert t.is_contiguous() and t.data_ptr() % 16 == 2 and not S._aligned(t)
    c = S._rows16(t)
    assert c.data_ptr() % 16 == 0 and c.is_contiguous() and c.shape == t.shape
    one = torch.as_strided(buf, (1, 4, 64), (261, 64, 1))
    assert S._aligned(one) and S._rows16(one) is one
    d = S._token_desc(one)
    assert (d.stride_b, d.stride_h, d.stride_n) == (0, 64, 0)
    assert S._token_desc(torch.as_strided(buf, (3, 1, 64), (64, 3, 1))).stride_h == 0
    page = torch.as_strided(buf, (1, 1, 4, 64), (3, 5, 64, 1))
    assert S._aligned(page)
    for hnd, want in ((True, (0, 0, 64)), (False, (0, 64, 0))):
        d = S._cache_desc(page, hnd)
        assert (d.stride_b, d.stride_h, d.stride_n) == want
    assert not S._aligned(torch.as_strided(buf, (2, 4, 64), (260, 64, 1)))
    assert not S._aligned(torch.as_strided(buf, (2, 4, 64), (256, 64, 2)))
    assert S._aligned(torch.zeros(0, 4, 64)) and S._aligned(torch.zeros(3, 0, 64))
