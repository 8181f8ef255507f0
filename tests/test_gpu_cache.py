"""Writing to the paged cache and reading it back, against 64-bit restatements.

Codes are compared with the nearest e4m3 value of the exact quotient: equal, except where the
quotient lies within fp32's error (2^-22 of it) of the midpoint of two codes; scales within one
fp32 step."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    _abi.load_library()
    return torch.device("cuda", 0)


def _check_codes(codes, scales, x):
    """codes [rows, dim] (e4m3) and scales [rows] of exact rows x."""
    expect, expect_scale = ref.quantise(x.double())
    assert ((scales.double() - expect_scale).abs() <= 2.0 ** -23 * expect_scale).all()
    quotient = x.double() * 448.0 / x.double().abs().amax(-1, keepdim=True).clamp(min=ref.FLOOR)
    step = ref.e4m3_step(quotient)
    tie = ((quotient / step) % 1.0 - 0.5).abs() * step <= 2.0 ** -22 * quotient.abs()
    got = codes.float().double()
    off = got != expect
    assert (off <= tie).all()
    assert ((got - expect).abs() <= step)[off].all()


def _setup(dev, lengths, new, heads, dim, size, dtype, cache_dtype, seed, layout="heads"):
    gen = torch.Generator().manual_seed(seed)
    table, pages = ref.page_table(lengths, size, dev, gen)
    cache = ref.make_cache(pages, size, heads, dim, cache_dtype, dev, gen, fill=-3.0, layout=layout)
    x = torch.randn(sum(new), 2, heads, dim, generator=gen) * torch.exp(2 * torch.randn(sum(new), 2, heads, 1, generator=gen))
    return table, cache, x.to(dtype).to(dev)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,size,lengths,new", [
    (1, 1, [1], [1]),
    (8, 16, [1, 16, 17, 33, 500], [1, 1, 1, 1, 1]),
    (3, 5, [20, 4, 9], [20, 0, 7]),
    (8, 64, [300, 3], [300, 1]),
])
def test_append(dev, dtype, cache_dtype, dim, heads, size, lengths, new):
    """Every new token lands in its slot, quantised; every other slot keeps its bytes."""
    table, cache, x = _setup(dev, lengths, new, heads, dim, size, dtype, cache_dtype, dim + heads)
    before = [t.clone() if t is not None else None for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)
    tokens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    uniform = len(set(new)) == 1
    cache.append(x[:, 0], x[:, 1], table, tokens, cu_seqlens=None if uniform else cu)
    assert cache.device_error() == 0
    touched = torch.zeros(cache.keys.shape[:1] + cache.keys.shape[2:3], dtype=torch.bool, device=dev)
    for b, length in enumerate(lengths):
        position = torch.arange(length - new[b], length, device=dev)
        page, slot = table[b].long()[position // size], position % size
        touched[page, slot] = True
        rows = x[sum(new[:b]):sum(new[:b + 1])]
        for j, (data, scales) in enumerate(((cache.keys, cache.key_scales), (cache.values, cache.value_scales))):
            if cache_dtype == E4M3:
                codes = data.view(torch.uint8)[page, :, slot].view(E4M3)
                _check_codes(codes.reshape(-1, dim), scales[page, :, slot].reshape(-1), rows[:, j].reshape(-1, dim))
            else:
                assert torch.equal(data[page, :, slot], rows[:, j])
    keep = ~touched[:, None].expand(cache.keys.shape[:3])
    for old, now in zip(before, (cache.keys, cache.values, cache.key_scales, cache.value_scales)):
        if old is not None:
            view = (lambda t: t.view(torch.uint8)) if old.dtype == E4M3 else (lambda t: t)
            assert torch.equal(view(old)[keep], view(now)[keep])


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("layout", ["slots", "padded"])
def test_append_and_gather_with_strides(dev, dtype, cache_dtype, layout):
    """Caches of other layouts, keys and values as slices of a fused projection."""
    lengths, new = [40, 21], [40, 21]
    table, cache, x = _setup(dev, lengths, new, 4, 128, 16, dtype, cache_dtype, 3, layout=layout)
    plain = ref.make_cache(cache.keys.size(0), 16, 4, 128, cache_dtype, dev, None, fill=-3.0)
    tokens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 40, 61], dtype=torch.int32, device=dev)
    fused = torch.zeros(61, 10, 128, dtype=dtype, device=dev)
    fused[:, 2:6], fused[:, 6:] = x[:, 0], x[:, 1]
    cache.append(fused[:, 2:6], fused[:, 6:], table, tokens, cu_seqlens=cu)
    plain.append(x[:, 0].contiguous(), x[:, 1].contiguous(), table, tokens, cu_seqlens=cu)
    for a, b in zip(cache.gather(table, cu, 61), plain.gather(table, cu, 61)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,size,lengths", [(1, 1, [1]), (8, 16, [0, 1, 16, 17, 0, 700, 0]), (3, 5, [23, 5, 4]), (2, 128, [1000])])
def test_gather(dev, dtype, cache_dtype, dim, heads, size, lengths):
    """Code * scale, rounded once; requests of no tokens among the others."""
    gen = torch.Generator().manual_seed(dim)
    table, pages = ref.page_table(lengths, size, dev, gen)
    cache = ref.make_cache(pages, size, heads, dim, cache_dtype, dev, gen)
    held = ref.fill_cache(cache, table, lengths, gen)
    starts = torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32, device=dev)
    got = cache.gather(table, starts, sum(lengths), dtype=dtype)
    assert cache.device_error() == 0
    for j in range(2):
        assert got[j].dtype == dtype
        # fp64 to the output type directly: one rounding (code * scale is exact in fp64)
        expect = torch.cat([pair[j] for pair in held])
        bound = expect.abs() * (1.01 * ref.EPS[dtype]) + ref.TINY[dtype] * 1.01
        assert ((got[j].double() - expect).abs() <= bound).all()


def test_a_rows_largest_value_survives(dev):
    """The largest magnitude of a row is code 448 exactly: read back within fp32 rounding of it."""
    table, cache, x = _setup(dev, [64], [64], 4, 128, 16, BF16, E4M3, 1)
    tokens = torch.tensor([64], dtype=torch.int32, device=dev)
    cache.append(x[:, 0], x[:, 1], table, tokens)
    assert (cache.keys.float().abs().amax(-1)[table[0, :4].long()] == 448.0).all()


@pytest.mark.parametrize("row,codes_nan,scale", [
    ([0.0], False, 2.0 ** -60 / 448), ([-0.0], False, 2.0 ** -60 / 448), ([1e-30], False, 2.0 ** -60 / 448),
    ([math.inf, 1.0], None, math.inf), ([math.nan, 1.0], True, math.nan), ([-math.inf, math.nan], True, math.nan),
    ([3e38], False, None), ([2.0 ** -59], False, 2.0 ** -59 / 448)])
def test_rows_at_the_edges(dev, row, codes_nan, scale):
    """Zeros and tiny rows stay finite; infinities and NaN make their row NaN when read back."""
    table, cache, x = _setup(dev, [3], [3], 2, 64, 16, BF16, E4M3, 2)
    x[1] = 0.0
    x[1, :, :, :len(row)] = torch.tensor(row, device=dev).to(BF16)
    tokens = torch.tensor([3], dtype=torch.int32, device=dev)
    cache.append(x[:, 0], x[:, 1], table, tokens)
    keys, values = cache.gather(table, torch.tensor([0, 3], dtype=torch.int32, device=dev), 3)
    for got, want in ((keys, x[:, 0]), (values, x[:, 1])):
        assert torch.isfinite(got[[0, 2]]).all()
        if codes_nan is False:
            assert (got[1].float() - want[1].float()).abs().max() <= max(2.0 ** -4 * abs(row[0]), 2.0 ** -60)
        else:
            assert torch.isnan(got[1]).all()
    page, slot = int(table[0, 0]), 1
    if scale is not None:
        got = cache.key_scales[page, :, slot]
        want = torch.full_like(got, scale)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and (torch.isnan(got) | (got == want) | ((got - want).abs() <= 2.0 ** -23 * want)).all()


def test_positions_before_the_start_are_skipped(dev):
    """More new tokens than the request's length: the ones at negative positions go nowhere."""
    table, cache, x = _setup(dev, [2, 5], [5, 5], 2, 64, 4, BF16, BF16, 4)
    cache.append(x[:, 0], x[:, 1], table, torch.tensor([2, 5], dtype=torch.int32, device=dev))
    keys, _ = cache.gather(table, torch.tensor([0, 2, 7], dtype=torch.int32, device=dev), 7)
    assert torch.equal(keys, torch.cat((x[3:5, 0], x[5:, 0]))) and cache.device_error() == 0


def test_rejected_drafts_are_overwritten(dev):
    """Lengths follow the accepted counts on the device: the next append overwrites the rest."""
    table, cache, x = _setup(dev, [12, 12], [8, 8], 2, 64, 4, BF16, E4M3, 5)
    lengths = torch.tensor([8, 8], dtype=torch.int32, device=dev)
    cache.append(x[:, 0], x[:, 1], table, lengths)
    accepted = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    lengths = lengths - 4 + accepted + 1 + 1  # one more token each
    again = x[[0, 8]] * 2
    cache.append(again[:, 0], again[:, 1], table, lengths)
    starts = torch.tensor([0, 6, 15], dtype=torch.int32, device=dev)
    keys, _ = cache.gather(table, starts, 15, dtype=BF16)
    assert torch.equal(keys[5], keys[0] * 2) and torch.equal(keys[14], keys[6] * 2)


@pytest.mark.parametrize("cache_dtype", [BF16, E4M3])
def test_offsets_past_32_bits(dev, cache_dtype):
    from sonic_sampler_b200.interface import PagedCache

    pages = 2 ** 32 // (128 * 8 * 64 * (1 if cache_dtype == E4M3 else 2)) + 8
    keys, values = (torch.empty(pages, 8, 64, 128, dtype=cache_dtype, device=dev) for _ in range(2))
    scales = [torch.empty(pages, 8, 64, device=dev) if cache_dtype == E4M3 else None for _ in range(2)]
    big = PagedCache(keys, values, *scales)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(100, 2, 8, 128, generator=gen).to(BF16).to(dev)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    small = ref.make_cache(2, 64, 8, 128, cache_dtype, dev, gen)
    tokens, starts = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([100], [0, 100]))
    big.append(x[:, 0], x[:, 1], table, tokens)
    small.append(x[:, 0], x[:, 1], torch.tensor([[1, 0]], dtype=torch.int32, device=dev), tokens)
    for a, b in zip(big.gather(table, starts, 100), small.gather(torch.tensor([[1, 0]], dtype=torch.int32, device=dev), starts, 100)):
        assert torch.equal(a, b)


def test_pages_outside_the_cache_are_skipped_and_reported(dev):
    from sonic_sampler_b200 import _abi

    table, cache, x = _setup(dev, [30, 30], [30, 30], 2, 64, 16, BF16, BF16, 6)
    tokens = torch.tensor([30, 30], dtype=torch.int32, device=dev)
    starts = torch.tensor([0, 30, 60], dtype=torch.int32, device=dev)
    before = cache.keys.clone()
    for bad in (-1, cache.keys.size(0), 2 ** 31 - 1):
        broken = table.clone()
        broken[1, 1] = bad
        cache.keys.copy_(before)
        cache.append(x[:, 0], x[:, 1], broken, tokens)
        assert cache.device_error() == _abi.DEVICE_ERR_PAGE and cache.device_error() == 0
        keys, _ = cache.gather(broken, starts, 60)
        assert cache.device_error() == _abi.DEVICE_ERR_PAGE
        assert torch.equal(keys[:46], x[:46, 0]) and not keys[46:].any()
    # a length past the page table's row
    cache.append(x[:, 0], x[:, 1], table[:, :1], tokens)
    assert cache.device_error() == _abi.DEVICE_ERR_PAGE


def test_rows_outside_every_request(dev):
    """Output rows that belong to no request are zeros; token rows that belong to none are not written."""
    table, cache, x = _setup(dev, [10], [10], 2, 64, 16, BF16, BF16, 7)
    tokens = torch.tensor([10], dtype=torch.int32, device=dev)
    wide = torch.cat((x, x))
    cache.append(wide[:, 0], wide[:, 1], table, tokens, cu_seqlens=torch.tensor([0, 10], dtype=torch.int32, device=dev))
    keys, _ = cache.gather(table, torch.tensor([2, 12], dtype=torch.int32, device=dev), 15)
    assert torch.equal(keys[2:12], x[:, 0]) and not keys[:2].any() and not keys[12:].any()


def test_streams_and_graphs(dev):
    table, cache, x = _setup(dev, [64], [64], 2, 64, 16, BF16, E4M3, 8)
    tokens, starts = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([64], [0, 64]))
    cache.append(x[:, 0], x[:, 1], table, tokens)
    expect = cache.gather(table, starts, 64)
    cache.keys.view(torch.uint8).fill_(0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.append(x[:, 0], x[:, 1], table, tokens)
        got = cache.gather(table, starts, 64)
    stream.synchronize()
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])
    cache.keys.view(torch.uint8).fill_(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(x[:, 0], x[:, 1], table, tokens)
        cache.gather(table, starts, 64, keys=got[0], values=got[1])
    got[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])


def test_refusals(dev):
    from sonic_sampler_b200 import _abi
    from sonic_sampler_b200.interface import PagedCache

    table, cache, x = _setup(dev, [10], [10], 2, 64, 16, BF16, BF16, 9)
    tokens, starts = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([10], [0, 10]))
    good = dict(keys=x[:, 0], values=x[:, 1], page_table=table, lengths=tokens)

    def refuse(message, **change):
        with pytest.raises(ValueError, match=message):
            cache.append(**{**good, **change})

    refuse("keys", keys=x[:, 0, :1])
    refuse("same number", keys=x[:5, 0])
    refuse("both be", keys=x[:, 0].half())
    refuse("of the cache's dtype", keys=x[:, 0].half(), values=x[:, 1].half())
    refuse("CUDA tensors only", keys=x[:, 0].cpu())
    refuse("must be on", values=x[:, 1].cpu())
    refuse("lengths", lengths=tokens.long())
    refuse("page_table", page_table=table.long())
    refuse("cu_seqlens", cu_seqlens=tokens)
    odd = torch.empty(10 * 2 * 64 + 8, dtype=BF16, device=dev)
    refuse("16-byte", keys=odd[1:1281].view(10, 2, 64))
    with pytest.raises(ValueError, match="starts"):
        cache.gather(table, starts.long(), 10)
    with pytest.raises(ValueError, match="dtype"):
        cache.gather(table, starts, 10, dtype=F16)
    with pytest.raises(ValueError, match="needs key_scales"):
        PagedCache(cache.keys.to(E4M3), cache.values.to(E4M3))
    with pytest.raises(ValueError, match="only a float8"):
        PagedCache(cache.keys, cache.values, torch.zeros(1, device=dev), torch.zeros(1, device=dev))
    with pytest.raises(ValueError, match="share strides"):
        PagedCache(cache.keys, cache.values.transpose(1, 2).contiguous().transpose(1, 2))
    small = PagedCache.allocate(2, 4, 1, 96, device=dev)
    with pytest.raises(_abi.SonicError, match="head_dim"):
        small.append(x[:1, 0, :1].repeat(1, 1, 2)[..., :96], x[:1, 0, :1].repeat(1, 1, 2)[..., :96], table[:, :1], tokens)
