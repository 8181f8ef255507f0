"""Sizes past 32 bits at the argument builders: refused, or (a window) as wide as any request, never taken
modulo 2^32. No memory behind them: strides of zero."""

from __future__ import annotations

import pytest
import torch

from sonic_sampler_b200 import ops
from sonic_sampler_b200.interface import PagedCache, ResidualNorm

BF16, I32 = torch.bfloat16, torch.int32
HUGE = 2 ** 32 + 3
CPU = torch.device("cpu")


def _rows(*shape):
    return torch.zeros(shape[-1], dtype=BF16).expand(*shape)


def test_norm_rows():
    norm = ResidualNorm(torch.ones(1, dtype=BF16))
    x = _rows(HUGE, 1)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.residual_norm_args(norm.template, x, norm.weight, None, None, x, None)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.residual_norm_args(norm.template, x[: 2 ** 31], norm.weight, None, None, x[: 2 ** 31], None)


def test_tokens():
    cache = PagedCache.allocate(1, 16, 1, 64, device="cpu")
    x, table = _rows(HUGE, 1, 64), torch.zeros(1, 1, dtype=I32)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.cache_append_args(cache.struct, x, x, table, torch.zeros(1, dtype=I32), cu_seqlens=None, flags=0, error=None, device=CPU)
    template = ops.paged_attention_template(1, 64, 0)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.paged_attention_args(template, cache.struct, x, table, torch.zeros(1, dtype=I32), cu_seqlens=None, max_tokens=0, window=0,
                                 scale=None, out=x, logsumexp=False, workspace=torch.zeros(1, dtype=torch.uint8), device=CPU)


def test_a_wide_window_hides_nothing():
    cache = PagedCache.allocate(1, 16, 1, 64, device="cpu")
    x, table = _rows(1, 1, 64), torch.zeros(1, 1, dtype=I32)
    template = ops.paged_attention_template(1, 64, 0)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32, HUGE, 2 ** 70):
        a, _, _ = ops.paged_attention_args(template, cache.struct, x, table, torch.zeros(1, dtype=I32), cu_seqlens=None, max_tokens=0,
                                           window=window, scale=None, out=x, logsumexp=False,
                                           workspace=torch.zeros(1, dtype=torch.uint8), device=CPU)
        assert a.window == 2 ** 31 - 1


def test_a_lookahead_of_32_bits():
    from sonic_sampler_b200.interface import PagedAttention

    with pytest.raises(ValueError, match="lookahead"):
        PagedAttention.initialize(1, 1, 64, lookahead=2 ** 31 - 1)
