"""The residual norm on rows narrower than a warp's loads, several of which share a warp: row counts
around its multiples, against the 64-bit restatement and against the same rows one by one."""

from __future__ import annotations

import pytest
import torch

from decode_reference import E4M3
from test_gpu_norm import BF16, F16, F32, _check, _inputs, dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out,group", [(None, None), (E4M3, None), (E4M3, 128)])
@pytest.mark.parametrize("hidden", [8, 32, 56, 64, 72, 120, 128, 136, 256])
@pytest.mark.parametrize("rows", [1, 3, 4, 15, 17, 1000])
def test_narrow_rows(dev, dtype, out, group, hidden, rows):  # noqa: F811
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, rows, hidden, dtype, rows + hidden)
    norm = ResidualNorm(weight, eps=1e-5, dtype=out, group=group)
    y, scales, r = norm(x, residual)
    _check(y, scales, r, x, residual, weight, 1e-5, group)
    y, scales, r = norm(x)
    _check(y, scales, r, x, None, weight, 1e-5, group)


@pytest.mark.parametrize("group", [None, 128])
def test_a_row_does_not_see_its_neighbours(dev, group):  # noqa: F811
    """An infinity, a NaN and huge values in one row of a shared warp leave the others as they are,
    bit for bit, and nothing is written past the rows."""
    from sonic_sampler_b200.interface import ResidualNorm

    for hidden in (64, 128):
        x, residual, weight = _inputs(dev, 9, hidden, BF16, hidden)
        norm = ResidualNorm(weight, dtype=E4M3, group=group)
        want = norm(x, residual)
        x[4, 3], x[6, 5], x[1] = float("nan"), float("inf"), 3e38
        buffers = [torch.full((12, t.size(1)), 7.0, device=dev).to(t.dtype) for t in want]
        got = norm(x, residual, out=buffers[0][:9], scales=buffers[1][:9], residual_out=buffers[2][:9])
        for g, w, b in zip(got, want, buffers):
            for row in (0, 2, 3, 5, 7, 8):
                assert torch.equal(g[row].view(torch.uint8), w[row].view(torch.uint8))
            assert (b[9:].float() == 7.0).all()
