"""What the build takes as up to date."""

from __future__ import annotations

import sysconfig

import torch

from sonic_sampler_b200 import build


def test_the_module_is_kept_by_torch_and_interpreter():
    assert torch.__version__ in build.calls_path().name and sysconfig.get_config_var("SOABI") in build.calls_path().name


def test_a_change_of_the_flags_makes_everything_stale(tmp_path):
    """build.py holds the compilers' flags: what is older than it is built again, as its objects are."""
    import os
    from pathlib import Path

    out, source = tmp_path / "out.so", tmp_path / "source.cu"
    out.touch()
    source.touch()
    written = Path(build.__file__).stat().st_mtime
    os.utime(source, (written - 200, written - 200))
    os.utime(out, (written - 100, written - 100))
    assert build.stale(out, [source])
    os.utime(out, (written + 100, written + 100))
    assert not build.stale(out, [source])
    os.utime(source, (written + 200, written + 200))
    assert build.stale(out, [source])
