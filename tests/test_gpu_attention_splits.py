"""How the paged attention's work is split and joined: page tables wider than the lengths (equal shares
of all requests' tiles, cut anywhere) and tight ones (a fixed number of warps a unit, from one to a
cluster of CTAs), for every number of query columns, against the 64-bit restatement."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from test_gpu_attention import BF16, E4M3, F16, _case, _check, dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def _check_wide(dev, lengths, new, q_heads, kv_heads, dim, dtype, cache_dtype, width, *, window=None, seed=0):  # noqa: F811
    """_check with a page table of `width` pages a row, the ones behind the lengths outside the cache."""
    from sonic_sampler_b200.interface import PagedAttention

    table, cache, held, q, first = _case(dev, lengths, new, q_heads, kv_heads, dim, 16, dtype, cache_dtype, seed)
    wide = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32, device=dev)
    wide[:, : table.size(1)] = table
    for b, n in enumerate(lengths):  # (a tight table's padding may hold pages of other requests)
        wide[b, -(-n // 16) :] = 1 << 30
    attention = PagedAttention.initialize(q_heads, kv_heads, dim, lookahead=max(new) - 1)
    cu = torch.tensor(first + [sum(new)], dtype=torch.int32, device=dev)
    out, lse = attention(q, cache, wide, torch.tensor(lengths, dtype=torch.int32, device=dev), cu_seqlens=cu, window=window,
                         logsumexp=True)
    expect, bound, expect_lse, lse_bound = ref.attention(q, held, lengths, new, first, kv_heads, window=window, scale=None,
                                                         weight_eps=ref.EPS[F16 if cache_dtype == E4M3 else dtype], out_dtype=dtype)
    assert attention.device_error() == 0
    assert not torch.isnan(out).any() and ((out.double() - expect).abs() <= bound).all()
    empty = torch.isinf(expect_lse)
    assert torch.equal(empty, lse == -math.inf)
    assert ((lse.double() - expect_lse).abs() <= lse_bound)[~empty].all()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,new", [(1, 1), (8, 1), (3, 5), (8, 2), (8, 3), (5, 5), (8, 4), (7, 4), (8, 5), (16, 5)])
def test_equal_shares_at_every_number_of_columns(dev, dtype, cache, dim, group, new):  # noqa: F811
    """One to four column tiles, full and partly filled, and several row tiles; long and short units
    next to each other, empty ones and requests shorter than their queries between them."""
    lengths = [900, 3, 0, 64, 129, 1500, 17, 1, 333]
    _check_wide(dev, lengths, [new, 1, 1, new, 1, new, new, new, 1], 2 * group, 2, dim, dtype, cache, 20000, seed=group + new)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("window", [1, 40, 700])
def test_equal_shares_with_a_window(dev, cache, window):  # noqa: F811
    _check_wide(dev, [900, 3, 0, 64, 2500], [4, 4, 1, 2, 4], 16, 2, 128, BF16, cache, 300000, window=window, seed=window)


@pytest.mark.parametrize("cache", [F16, E4M3])
@pytest.mark.parametrize("new", [1, 4, 6, 8])
def test_a_unit_of_many_ctas_is_joined_in_two_levels(dev, cache, new):  # noqa: F811
    """One kv head and 50021 keys: more than 12 CTAs have a part, with one to four column tiles."""
    _check(dev, [50021, 130], [new, 1], 4, 1, 64, 64, F16, cache, seed=new)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("new", [1, 3, 5, 8])
@pytest.mark.parametrize("requests,longest", [(300, 60), (150, 600), (60, 700), (30, 900), (12, 1500), (1, 2000)])
def test_fixed_numbers_of_warps(dev, cache, new, requests, longest):  # noqa: F811
    """From a warp a unit to clusters of eight CTAs; lengths from none to the longest, so that
    some of a unit's warps have nothing to do."""
    lengths = [longest - (longest * 7 * b // max(requests, 2)) % (longest + 1) for b in range(requests)]
    _check(dev, lengths, [new] * requests, 8, 2, 64, 16, BF16, cache, ragged=False, seed=requests)


def test_splits_follow_the_lengths_alone(dev):  # noqa: F811
    """The same requests with their pages in other places, on the same path: the same bits."""
    from sonic_sampler_b200.interface import PagedAttention

    lengths = [700, 12, 0, 3000]
    table, cache, _, q, _ = _case(dev, lengths, [1] * 4, 8, 2, 128, 16, BF16, BF16, 1)
    attention = PagedAttention.initialize(8, 2, 128)
    tokens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = attention(q, cache, table, tokens)
    order = torch.randperm(cache.keys.size(0), generator=torch.Generator().manual_seed(2)).to(dev)
    cache.keys.copy_(cache.keys[order])
    cache.values.copy_(cache.values[order])
    where = torch.empty_like(order)
    where[order] = torch.arange(order.numel(), device=dev)
    moved = where[table.long().clamp(0, order.numel() - 1)].to(torch.int32)
    assert torch.equal(attention(q, cache, moved, tokens), want)
