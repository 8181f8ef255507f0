"""What the build takes as up to date."""

from __future__ import annotations

import sysconfig

import torch

from sonic_sampler_b200 import build


def test_the_module_is_kept_by_torch_and_interpreter():
    assert torch.__version__ in build.calls_path().name and sysconfig.get_config_var("SOABI") in build.calls_path().name
