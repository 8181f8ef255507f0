"""Value scales of an e4m3 cache far from ordinary ones: zero (fresh pages, an engine's own zero rows),
tiny and large, on every way that a request's keys are split and joined.

Bounds. Weights are rounded to fp16 with their value scale on, the largest as 2^6 to 2^14: relative 2^-11,
and below fp16's smallest normal number within 2^-25. Where ordinary scales lead, that is the bound of
ordinary caches. Where keys of a scale of zero, or below 2^-80, hold nearly all of the weight, the
weights' sum is at least 2^90, and n keys of codes up to 448 are off by n * 448 * 2^-25 / 2^90. A result
below bf16's smallest normal number is off by half of its smallest step, 2^-134."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from test_gpu_attention import BF16, E4M3, F16, _case, dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def _scaled(dev, lengths, new, q_heads, kv_heads, dim, factors, seed, width=0):  # noqa: F811
    """A case whose value scales are multiplied by factors[b] [length, kv_heads]; a page table of
    `width` pages a row picks the way of equal shares."""
    table, cache, held, q, first = _case(dev, lengths, new, q_heads, kv_heads, dim, 16, BF16, E4M3, seed)
    for b, (n, factor) in enumerate(zip(lengths, factors)):
        position = torch.arange(n, device=dev)
        page, slot = table[b].long()[position // 16], position % 16
        cache.value_scales[page, :, slot] = (cache.value_scales[page, :, slot].double() * factor.to(dev)).float()
        keys, values = held[b]
        codes = cache.values.view(torch.uint8)[page, :, slot].view(E4M3).double()
        held[b] = (keys, codes * cache.value_scales[page, :, slot].double()[..., None])
    if width:
        wide = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32, device=dev)
        for b, n in enumerate(lengths):
            wide[b, : -(-n // 16)] = table[b, : -(-n // 16)]
        table = wide
    return table, cache, held, q, first


def _attend(dev, table, cache, q, lengths, new, first, q_heads, kv_heads, dim):  # noqa: F811
    from sonic_sampler_b200.interface import PagedAttention

    attention = PagedAttention.initialize(q_heads, kv_heads, dim, lookahead=max(new) - 1)
    cu = torch.tensor(first + [sum(new)], dtype=torch.int32, device=dev)
    out, lse = attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=dev), cu_seqlens=cu, logsumexp=True)
    assert attention.device_error() == 0
    return out, lse


def _expect(q, held, lengths, new, first, kv_heads):
    """(out, bound, log-sum-exp, bound)."""
    expect, bound, lse, lse_bound = ref.attention(q, held, lengths, new, first, kv_heads, weight_eps=ref.EPS[F16], out_dtype=BF16)
    keys = torch.tensor(lengths, device=q.device).repeat_interleave(torch.tensor(new, device=q.device))
    return expect, bound + (keys * 448.0 * 2.0 ** -115 + 2.0 ** -134).view(-1, 1, 1), lse, lse_bound


def _check(dev, lengths, new, q_heads, kv_heads, dim, factors, seed, width=0):  # noqa: F811
    table, cache, held, q, first = _scaled(dev, lengths, new, q_heads, kv_heads, dim, factors, seed, width)
    out, lse = _attend(dev, table, cache, q, lengths, new, first, q_heads, kv_heads, dim)
    expect, bound, expect_lse, lse_bound = _expect(q, held, lengths, new, first, kv_heads)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert ((lse.double() - expect_lse).abs() <= lse_bound).all()
    assert ((out.double() - expect).abs() <= bound).all()


def _ones(lengths, kv_heads):
    return [torch.ones(n, kv_heads, dtype=torch.float64) for n in lengths]


#: tight tables: from one warp a request to a cluster of CTAs; wide ones: equal shares, long requests cut
WAYS = [([40] * 300, 0), ([33, 700, 40, 5], 0), ([900, 41, 33, 6000], 30000), ([50021, 130], 0)]


@pytest.mark.parametrize("group,new,dim", [(4, 1, 128), (8, 3, 128), (8, 4, 64), (8, 2, 256)])
@pytest.mark.parametrize("way", range(len(WAYS)))
@pytest.mark.parametrize("where", ["all", "first", "middle", "half", "some"])
def test_scales_of_zero(dev, group, new, dim, way, where):  # noqa: F811
    """A key whose value scale is zero weighs in the sum and adds nothing: over the whole of every
    request, its first keys (a warp's first tiles), 40 in its middle, its first half (whole shares of
    warps), every third one."""
    lengths, width = WAYS[way]
    if way == 0:
        lengths = lengths[: 300 if new == 1 else 75]
    factors = _ones(lengths, 2)
    for f in factors:
        n = f.size(0)
        f[{"all": slice(None), "first": slice(0, min(40, n - 1)), "middle": slice(n // 2, n // 2 + 40), "half": slice(0, n // 2),
           "some": slice(0, None, 3)}[where]] = 0.0
    _check(dev, lengths, [new] * len(lengths), 2 * group, 2, dim, factors, seed=way, width=width)


@pytest.mark.parametrize("power", [-140, -120, -100, -69, -60, 60, 100])
@pytest.mark.parametrize("way", range(len(WAYS)))
def test_scales_tiny_and_large(dev, power, way):  # noqa: F811
    """Whole requests at 2^-140 to 2^100 of the ordinary, at 2^-60 with zeros between. Below 2^-80 the results
    fade; the log-sum-exps do not."""
    lengths, width = WAYS[way]
    factors = [f * 2.0 ** power for f in _ones(lengths, 2)]
    if power == -60:
        for f in factors:
            f[::5] = 0.0
    _check(dev, lengths, [1] * len(lengths), 8, 2, 128, factors, seed=way, width=width)


@pytest.mark.parametrize("way", range(len(WAYS)))
def test_scales_of_either_sign(dev, way):  # noqa: F811
    """A row stands for code * scale, whatever the scale's sign."""
    lengths, width = WAYS[way]
    factors = _ones(lengths, 2)
    for f in factors:
        f[::3] = -1.0
    _check(dev, lengths, [1] * len(lengths), 8, 2, 128, factors, seed=way, width=width)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("way", range(len(WAYS)))
@pytest.mark.parametrize("at", [0, 20, -1])
def test_log_sum_exps_do_not_depend_on_bad_value_scales(dev, bad, way, at):  # noqa: F811
    """A value row that is not finite, the first, one of a later request's first keys or the newest: the
    output is not finite where it is seen, the log-sum-exp is that of the keys."""
    lengths, width = WAYS[way]
    new = [2] * len(lengths)
    factors = _ones(lengths, 2)
    table, cache, held, q, first = _scaled(dev, lengths, new, 8, 2, 128, factors, way, width)
    for b, n in enumerate(lengths):
        p = at % n
        cache.value_scales[table[b, p // 16].long(), :, p % 16] = bad
    out, lse = _attend(dev, table, cache, q, lengths, new, first, 8, 2, 128)
    expect, bound, expect_lse, lse_bound = _expect(q, held, lengths, new, first, 2)
    assert ((lse.double() - expect_lse).abs() <= lse_bound).all()
    for b, n in enumerate(lengths):
        rows = slice(first[b] + (at == -1), first[b] + 2)
        assert not torch.isfinite(out[rows]).any()
        if at == -1:  # the request's first query does not see its last key
            assert ((out[first[b]].double() - expect[first[b]]).abs() <= bound[first[b]]).all()
