"""Attention over the paged cache against its 64-bit restatement, at the sizes, masks and layouts
where it can go wrong. Every unwritten slot of the caches holds NaN, so a read past a mask shows."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    _abi.load_library()
    return torch.device("cuda", 0)


def _case(dev, lengths, new, q_heads, kv_heads, dim, page_size, dtype, cache_dtype, seed, layout="heads", scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    table, pages = ref.page_table(lengths, page_size, dev, gen)
    cache = ref.make_cache(pages, page_size, kv_heads, dim, cache_dtype, dev, gen, layout=layout)
    held = ref.fill_cache(cache, table, lengths, gen, scale=scale)
    q = (torch.randn(sum(new), q_heads, dim, generator=gen) * 1.5).to(dtype).to(dev)
    first = [sum(new[:b]) for b in range(len(new))]
    return table, cache, held, q, first


def _check(dev, lengths, new, q_heads, kv_heads, dim, page_size, dtype, cache_dtype, *, window=None, ragged=True, seed=0,
           layout="heads", scale=None, lookahead=None):
    from sonic_sampler_b200.interface import PagedAttention

    table, cache, held, q, first = _case(dev, lengths, new, q_heads, kv_heads, dim, page_size, dtype, cache_dtype, seed, layout)
    attention = PagedAttention.initialize(q_heads, kv_heads, dim, lookahead=max(new) - 1 if lookahead is None else lookahead)
    cu = torch.tensor(first + [sum(new)], dtype=torch.int32, device=dev) if ragged else None
    out, lse = attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=dev), cu_seqlens=cu, window=window,
                         scale=scale, logsumexp=True)
    weight_eps = ref.EPS[F16 if cache_dtype == E4M3 else dtype]
    expect, bound, expect_lse, lse_bound = ref.attention(q, held, lengths, new, first, kv_heads, window=window, scale=scale,
                                                         weight_eps=weight_eps, out_dtype=dtype)
    assert attention.device_error() == 0
    assert out.dtype == dtype and lse.dtype == torch.float32
    far = (out.double() - expect).abs() / bound
    assert not torch.isnan(out).any() and far.max() <= 1.0, far.max()
    empty = torch.isinf(expect_lse)
    assert torch.equal(empty, lse == -math.inf)
    assert ((lse.double() - expect_lse).abs() <= lse_bound)[~empty].all()
    return attention, q, cache, table, cu, out, lse


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (3, 1), (32, 2)])
def test_lengths_around_the_tiles(dev, dtype, cache, dim, q_heads, kv_heads):
    """One token a request, from an empty request over every boundary of a warp's tile and a step."""
    lengths = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 0, 700]
    _check(dev, lengths, [1] * len(lengths), q_heads, kv_heads, dim, 16, dtype, cache, ragged=False, seed=dim)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("page_size", [1, 5, 8, 16, 24, 64, 128])
def test_page_sizes(dev, dtype, cache, page_size):
    _check(dev, [130, 1, 311, 64], [1] * 4, 8, 2, 128, page_size, dtype, cache, ragged=False, seed=page_size)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [None, 1, 3, 70])
def test_several_tokens_a_request(dev, dtype, cache, dim, window):
    """Queries of one request see different keys; some requests are shorter than their queries, so
    that their first queries see none, and one has no query at all."""
    lengths, new = [66, 3, 0, 200, 16, 1, 129], [5, 5, 2, 1, 16, 3, 0]
    _check(dev, lengths, new, 8, 2, dim, 16, dtype, cache, window=window, seed=7)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new", [1, 2, 4, 5, 16])
@pytest.mark.parametrize("q_heads,kv_heads", [(5, 5), (14, 2), (16, 1), (64, 8)])
def test_head_layouts(dev, dtype, cache, new, q_heads, kv_heads):
    """Group sizes 1, 7, 16 and 8 with up to 256 query rows a key head: tiles of one and two rows of
    16, partly filled, and several tiles a unit."""
    _check(dev, [100, new, 333], [new] * 3, q_heads, kv_heads, 64, 16, dtype, cache, ragged=False, seed=new)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_a_wrong_lookahead_hint_changes_nothing(dev, dtype, cache):
    """More tokens than `lookahead + 1`: a prompt's chunk of 70 tokens beside a single one."""
    _check(dev, [150, 40], [70, 1], 8, 2, 128, 16, dtype, cache, lookahead=0, window=64, seed=3)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim,kv_heads,length", [(128, 8, 9001), (64, 1, 40011), (256, 2, 5003)])
def test_long_sequences_are_split_and_joined(dev, dtype, cache, dim, kv_heads, length):
    """Every CTA takes a part of a few units; their parts are joined through the workspace."""
    _check(dev, [length, 13], [1, 1], 4 * kv_heads, kv_heads, dim, 64, dtype, cache, ragged=False, seed=length)
    _check(dev, [length, 77], [2, 3], 4 * kv_heads, kv_heads, dim, 64, dtype, cache, window=length - 900, seed=length)


@pytest.mark.parametrize("requests", [1, 127, 128, 129, 700])
def test_many_requests(dev, requests):
    """More requests than threads scan, lengths of every size, several a CTA."""
    lengths = [(37 * b) % 211 for b in range(requests)]
    _check(dev, lengths, [1] * requests, 4, 1, 64, 16, BF16, BF16, ragged=False, seed=requests)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("layout", ["slots", "padded"])
def test_strided_caches(dev, dtype, cache, layout):
    _check(dev, [95, 240], [3, 1], 8, 2, 128, 16, dtype, cache, layout=layout, seed=5)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_strided_queries_and_outputs(dev, dtype, cache):
    """Queries as a slice of a fused projection, the output as a slice of a wider tensor."""
    attention, q, pages, table, cu, out, _ = _check(dev, [95, 240], [3, 1], 8, 2, 128, 16, dtype, cache, seed=6)
    lengths = torch.tensor([95, 240], dtype=torch.int32, device=dev)
    fused = torch.full((4, 12, 128), math.nan, dtype=dtype, device=dev)
    fused[:, 2:10] = q
    wide = torch.zeros(4, 10, 160, dtype=dtype, device=dev)
    attention(fused[:, 2:10], pages, table, lengths, cu_seqlens=cu, output=wide[:, 1:9, 16:144])
    assert torch.equal(wide[:, 1:9, 16:144], out)
    wide[:, 1:9, 16:144] = 0
    assert not wide.any()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("scale", [0.01, 3.0])
def test_scales_flat_and_sharp(dev, dtype, cache, scale):
    """Nearly uniform weights, and weights where one key takes all."""
    _check(dev, [333, 64], [1, 4], 8, 2, 128, 16, dtype, cache, scale=scale, seed=8)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_a_query_does_not_see_never_reaches_it(dev, dtype, cache, bad):
    """NaN or infinite keys and values of the newest token: the queries before it are untouched,
    and the one that sees it is NaN."""
    from sonic_sampler_b200.interface import PagedAttention

    lengths, new = [37, 64, 20], [4, 4, 4]
    table, pages, held, q, first = _case(dev, lengths, new, 8, 2, 128, 16, dtype, cache, 9)
    attention = PagedAttention.initialize(8, 2, 128, lookahead=3)
    tokens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    clean = attention(q, pages, table, tokens)
    for b, length in enumerate(lengths):
        page, slot = int(table[b, (length - 1) // 16]), (length - 1) % 16
        if cache == E4M3:
            pages.values.view(torch.uint8)[page, :, slot] = 0x7f
            pages.value_scales[page, :, slot] = bad
            pages.key_scales[page, :, slot] = bad
        else:
            pages.values[page, :, slot] = bad
            pages.keys[page, :, slot] = bad
    out, lse = attention(q, pages, table, tokens, logsumexp=True)
    for b in range(3):
        rows = slice(first[b], first[b] + 3)
        assert torch.equal(out[rows], clean[rows])
        assert torch.isfinite(lse[rows]).all()
        assert torch.isnan(out[first[b] + 3]).all()
    # and a window that has moved past the token
    for b, length in enumerate(lengths):
        page, slot = int(table[b, (length - 5) // 16]), (length - 5) % 16
        if cache == E4M3:
            pages.values.view(torch.uint8)[page, :, slot] = 0xff
        else:
            pages.values[page, :, slot] = -bad
    out = attention(q, pages, table, tokens, window=2)
    for b in range(3):
        # query 0 (position length - 4) sees the second token; queries 1 and 2 do not
        assert not torch.isfinite(out[first[b]]).any()
        assert torch.isfinite(out[first[b] + 1:first[b] + 3]).all()


def test_value_scales_of_any_size(dev):
    """e4m3 value rows whose scales span 60 binades: the weights keep their precision."""
    from sonic_sampler_b200.interface import PagedAttention

    lengths, new = [200], [1]
    table, pages, held, q, first = _case(dev, lengths, new, 4, 1, 128, 16, BF16, E4M3, 10)
    keys, values = held[0]
    factor = torch.exp2(torch.randint(-40, 20, (200, 1), generator=torch.Generator().manual_seed(1)).double()).to(dev)
    position = torch.arange(200, device=dev)
    page, slot = table[0].long()[position // 16], position % 16
    pages.value_scales[page, :, slot] *= factor.float()
    held = [(keys, values * factor[..., None])]
    attention = PagedAttention.initialize(4, 1, 128)
    out = attention(q, pages, table, torch.tensor(lengths, dtype=torch.int32, device=dev))
    expect, bound, _, _ = ref.attention(q, held, lengths, new, first, 1, weight_eps=ref.EPS[F16], out_dtype=BF16)
    assert ((out.double() - expect).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_any_size(dev, dtype):
    """Query rows far from 1 meet e4m3 keys as fp16: brought into its range row by row."""
    from sonic_sampler_b200.interface import PagedAttention

    lengths, new = [120], [1]
    table, pages, held, q, first = _case(dev, lengths, new, 8, 1, 64, 16, dtype, E4M3, 11)
    powers = torch.tensor([1.0, 2.0 ** -14, 2.0 ** -8, 2.0 ** 8, 2.0 ** 13 if dtype == F16 else 2.0 ** 60, 0.0, 2.0 ** -10, 1.0], device=dev)
    q = (q * powers[None, :, None]).to(dtype)
    scale = torch.where(powers > 0, 1.0 / powers.clamp(min=1e-30), 1.0)
    attention = PagedAttention.initialize(8, 1, 64)
    for h in range(8):  # a scale that gives every head ordinary scores
        out = attention(q, pages, table, torch.tensor(lengths, dtype=torch.int32, device=dev), scale=float(scale[h]) / 8.0)
        expect, bound, _, _ = ref.attention(q[:, h:h + 1], held, lengths, new, first, 1, scale=float(scale[h]) / 8.0,
                                            weight_eps=ref.EPS[F16], out_dtype=dtype)
        assert ((out[:, h:h + 1].double() - expect).abs() <= bound).all()


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_offsets_past_32_bits(dev, cache):
    """Pages whose first element lies beyond 2^32 bytes of the cache's start."""
    from sonic_sampler_b200.interface import PagedAttention, PagedCache

    dim, heads, size = 128, 8, 64
    pages = 2 ** 32 // (dim * heads * size * (1 if cache == E4M3 else 2)) + 40
    keys, values = (torch.empty(pages, heads, size, dim, dtype=cache, device=dev) for _ in range(2))
    scales = [torch.empty(pages, heads, size, device=dev) if cache == E4M3 else None for _ in range(2)]
    big = PagedCache(keys, values, *scales)
    gen = torch.Generator().manual_seed(12)
    lengths = [300, 129]
    table = (pages - 1 - torch.arange(10, dtype=torch.int32)).view(2, 5).to(dev)
    held = ref.fill_cache(big, table, lengths, gen)
    q = torch.randn(2, 16, dim, generator=gen).to(BF16).to(dev)
    out = PagedAttention.initialize(16, heads, dim)(q, big, table, torch.tensor(lengths, dtype=torch.int32, device=dev))
    expect, bound, _, _ = ref.attention(q, held, lengths, [1, 1], [0, 1], heads, weight_eps=ref.EPS[F16 if cache == E4M3 else BF16],
                                        out_dtype=BF16)
    assert ((out.double() - expect).abs() <= bound).all()


def test_calls_repeat_exactly_and_follow_a_captured_graph(dev):
    """The same call gives the same bits; a graph's replay follows lengths and pages on the device."""
    attention, q, cache, table, cu, out, lse = _check(dev, [1500, 3, 800], [1, 1, 1], 8, 2, 128, 16, BF16, BF16, seed=13)
    lengths = torch.tensor([1500, 3, 800], dtype=torch.int32, device=dev)
    static = torch.empty_like(out)
    for _ in range(5):
        attention(q, cache, table, lengths, output=static)
        assert torch.equal(static, attention(q, cache, table, lengths))
    shorter = torch.tensor([600, 2, 1], dtype=torch.int32, device=dev)
    expect = attention(q, cache, table, shorter)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention(q, cache, table, lengths, output=static)
    graph.replay()
    torch.cuda.synchronize()
    lengths.copy_(shorter)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(static, expect)


def test_on_another_stream(dev):
    attention, q, cache, table, cu, out, _ = _check(dev, [400, 90], [1, 1], 8, 2, 128, 16, BF16, E4M3, seed=14)
    lengths = torch.tensor([400, 90], dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = attention(q, cache, table, lengths)
    stream.synchronize()
    assert torch.equal(out, again)


def test_pages_and_lengths_outside_the_cache_are_reported(dev):
    """A bad page id or length is found on the device; the other requests' outputs stand."""
    from sonic_sampler_b200 import _abi

    attention, q, cache, table, cu, out, _ = _check(dev, [100, 50, 70], [1, 1, 1], 4, 1, 64, 16, BF16, BF16, seed=15)
    lengths = torch.tensor([100, 50, 70], dtype=torch.int32, device=dev)
    for bad in (-1, cache.keys.size(0), 2 ** 31 - 1):
        broken = table.clone()
        broken[1, 2] = bad
        got = attention(q, cache, broken, lengths)
        assert attention.device_error() == _abi.DEVICE_ERR_PAGE and attention.device_error() == 0
        assert torch.equal(got[[0, 2]], out[[0, 2]])
    for bad in (-3, table.size(1) * 16 + 1, 2 ** 31 - 1):
        got = attention(q, cache, table, torch.tensor([100, bad, 70], dtype=torch.int32, device=dev))
        assert attention.device_error() & _abi.DEVICE_ERR_PAGE
        assert torch.equal(got[[0, 2]], out[[0, 2]])
    assert torch.equal(attention(q, cache, table, lengths), out)


def test_nothing_to_do(dev):
    from sonic_sampler_b200.interface import PagedAttention

    attention, q, cache, table, cu, _, _ = _check(dev, [0, 0], [1, 1], 4, 1, 64, 16, BF16, BF16, seed=16)
    out = attention(q[:0], cache, table, torch.zeros(2, dtype=torch.int32, device=dev))
    assert out.shape == (0, 4, 64)


def test_refusals(dev):
    from sonic_sampler_b200 import _abi
    from sonic_sampler_b200.interface import PagedAttention

    attention, q, cache, table, cu, _, _ = _check(dev, [20, 30], [1, 1], 4, 1, 64, 16, BF16, BF16, seed=17)
    lengths = torch.tensor([20, 30], dtype=torch.int32, device=dev)
    good = dict(queries=q, cache=cache, page_table=table, lengths=lengths)

    def refuse(message, **change):
        with pytest.raises(ValueError, match=message):
            attention(**{**good, **change})

    refuse("queries", queries=q[:, :2])
    refuse("queries", queries=q.float())
    refuse("unit inner stride", queries=q.transpose(0, 2).contiguous().transpose(0, 2))
    refuse("cache's dtype", queries=q.half())
    refuse("CUDA tensors only", queries=q.cpu())
    refuse("page_table", page_table=table.long())
    refuse("page_table", page_table=table.cpu())
    refuse("lengths", lengths=lengths.long())
    refuse("lengths", lengths=lengths[:1])
    refuse("cu_seqlens", cu_seqlens=lengths)
    refuse("same number of tokens", queries=q[:1])
    refuse("window", window=0)
    refuse("output", output=torch.empty(2, 4, 64, dtype=F16, device=dev))
    refuse("finite", scale=math.nan)
    odd = torch.empty(2 * 4 * 64 + 8, dtype=BF16, device=dev)
    refuse("16-byte", queries=odd[1:513].view(2, 4, 64))
    refuse("8-byte", output=odd[1:513].view(2, 4, 64))
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        PagedAttention.initialize(5, 2, 64)
    with pytest.raises(ValueError, match="head_dim"):
        PagedAttention.initialize(4, 2, 96)
    attention.scratchpad = attention.scratchpad[:1024]
    with pytest.raises(_abi.SonicError, match="workspace"):
        attention(**good)
