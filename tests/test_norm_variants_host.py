"""The norm's kernels in the library are those that some row's width reaches."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from sonic_sampler_b200 import build

WIDEST = 32768


def test_no_variant_is_wider_than_the_widest_row():
    nm = shutil.which("nm")
    if not nm:
        pytest.skip("needs nm")
    names = subprocess.run([nm, "-C", str(build.build())], check=True, capture_output=True, text=True).stdout
    found = set(re.findall(r"norm_kernel<(\w+), (true|false), (true|false), (\d+), (\d+)>", names))
    assert found
    for dtype, _, vec, items, width in found:
        columns = int(width) * ((4 if dtype == "float" else 8) if vec == "true" else 4)
        # fewer items a lane reach the widest row with a CTA's 32 warps, or this many are needed
        assert int(items) <= 4 or int(items) // 2 * columns * 32 < WIDEST, (dtype, vec, items, width)
