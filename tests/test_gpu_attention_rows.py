"""Token rows of a call that belong to no request, as in a captured graph whose token count is padded:
before `cu_seqlens[0]` and from `cu_seqlens[-1]` on. They see no key: zeros, and a log-sum-exp of
-infinity, whatever their queries, and the output's memory, held."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from test_gpu_attention import BF16, E4M3, F16, _case, dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu

#: equal shares; fixed numbers of warps: a cluster of CTAs, one CTA, one warp a request and head
WAYS = [([900, 3, 0, 64, 2500], 20000), ([700], 0), ([600] * 30, 0), ([40] * 300, 0)]


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, E4M3)])
@pytest.mark.parametrize("way", range(len(WAYS)))
@pytest.mark.parametrize("before,after", [(0, 1), (1, 0), (0, 300), (37, 5)])
@pytest.mark.parametrize("strided", [False, True])
def test_rows_of_no_request_are_zero(dev, dtype, cache_dtype, way, before, after, strided):  # noqa: F811
    from sonic_sampler_b200.interface import PagedAttention

    lengths, width = WAYS[way]
    new = [1 + b % 2 for b in range(len(lengths))]
    table, cache, held, q, first = _case(dev, lengths, new, 8, 2, 64, 16, dtype, cache_dtype, 1)
    if width:
        wide = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32, device=dev)
        for b, n in enumerate(lengths):
            wide[b, : -(-n // 16)] = table[b, : -(-n // 16)]
        table = wide
    live = sum(new)
    padded = torch.full((before + live + after, 8, 64), math.nan, dtype=dtype, device=dev)
    padded[before:before + live] = q
    cu = torch.tensor([before + f for f in first] + [before + live], dtype=torch.int32, device=dev)
    attention = PagedAttention.initialize(8, 2, 64, lookahead=1)
    room = torch.full((before + live + after, 10, 72), 7.0, dtype=dtype, device=dev)
    given = room[:, 1:9, 8:] if strided else torch.full_like(padded, 7.0)
    out, lse = attention(padded, cache, table, torch.tensor(lengths, dtype=torch.int32, device=dev), cu_seqlens=cu, output=given,
                         logsumexp=True)
    assert out is given and attention.device_error() == 0
    expect, bound, expect_lse, lse_bound = ref.attention(q, held, lengths, new, first, 2, out_dtype=dtype,
                                                         weight_eps=ref.EPS[F16 if cache_dtype == E4M3 else dtype])
    inside = slice(before, before + live)
    assert ((out[inside].double() - expect).abs() <= bound).all()
    seen = torch.isfinite(expect_lse)
    assert torch.equal(seen, torch.isfinite(lse[inside]))
    assert ((lse[inside].double() - expect_lse).abs() <= lse_bound)[seen].all()
    for outside in (slice(0, before), slice(before + live, None)):
        assert (out[outside] == 0).all() and (lse[outside] == -math.inf).all()
    if strided:
        given.fill_(7.0)
        assert (room == 7.0).all()


@pytest.mark.parametrize("width", [1, 20000])
def test_no_request_has_a_row(dev, width):  # noqa: F811
    """Every request without new tokens, or without keys, in a call of padding."""
    from sonic_sampler_b200.interface import PagedAttention

    cache = ref.make_cache(4, 16, 2, 64, BF16, dev, torch.Generator().manual_seed(1))
    attention = PagedAttention.initialize(4, 2, 64)
    q = torch.randn(9, 4, 64, device=dev).to(BF16)
    table = torch.zeros(3, width, dtype=torch.int32, device=dev)
    for cu, lengths in (([0, 0, 0, 0], [5, 0, 1]), ([9, 9, 9, 9], [5, 0, 1]), ([4, 4, 4, 4], [0, 0, 0]), ([2, 3, 3, 7], [0, 0, 0])):
        given = torch.full_like(q, math.nan)
        out, lse = attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=dev),
                             cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev), output=given, logsumexp=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    assert attention.device_error() == 0
