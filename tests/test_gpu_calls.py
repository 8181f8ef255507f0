"""The two ways of a call from Python, the compiled one and the argument builders: the same outputs, bit
for bit, and the same errors; what the compiled one does not take goes on to the builders."""

from __future__ import annotations

import gc
import math

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


class NoCalls:
    """In place of the compiled module: everything goes to the builders."""

    norm = append = gather = attention = staticmethod(lambda *args: None)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    _abi.load_library()
    return torch.device("cuda", 0)


def _both(monkeypatch, call):
    """What `call()` gives by the compiled way, and by the builders."""
    from sonic_sampler_b200 import _abi

    compiled = call()
    with monkeypatch.context() as m:
        m.setattr(_abi, "_CALLS", NoCalls)
        built = call()
    return compiled, built


def _same(a, b):
    assert type(a) is type(b)
    if isinstance(a, tuple):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            _same(x, y)
    elif a is not None:
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.device == b.device
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out,group", [(None, None), (E4M3, None), (E4M3, 128)])
@pytest.mark.parametrize("rows,hidden", [(0, 64), (1, 1), (5, 200), (3, 257)])
def test_norm(dev, monkeypatch, dtype, out, group, rows, hidden):
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual = (torch.randn(rows, hidden + 3, device=dev).to(dtype)[:, :hidden] for _ in range(2))
    norm = ResidualNorm(torch.randn(hidden, device=dev).to(dtype), dtype=out, group=group)
    _same(*_both(monkeypatch, lambda: norm(x)))
    _same(*_both(monkeypatch, lambda: norm(x, residual)))
    _same(*_both(monkeypatch, lambda: norm(x.contiguous().view(1, rows, hidden))))
    _same(*_both(monkeypatch, lambda: norm(torch.nn.Parameter(x))))


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("ragged", [False, True])
def test_cache_and_attention(dev, monkeypatch, dtype, cache_dtype, ragged):
    from sonic_sampler_b200.interface import PagedAttention

    gen = torch.Generator().manual_seed(1)
    lengths = [40, 2, 7]
    table, pages = ref.page_table(lengths, 16, dev, gen)
    tokens = torch.tensor(lengths, dtype=I32, device=dev)
    starts = torch.tensor([0, 40, 42, 49], dtype=I32, device=dev)
    fused = torch.randn(49, 8, 64, generator=gen).to(dtype).to(dev)
    caches = []

    def write():
        caches.append(ref.make_cache(pages, 16, 2, 64, cache_dtype, dev, torch.Generator().manual_seed(2)))
        assert caches[-1].append(fused[:, 4:6], fused[:, 6:], table, tokens, starts) is caches[-1]

    _both(monkeypatch, write)
    for name in ("keys", "values", "key_scales", "value_scales"):
        _same(getattr(caches[0], name), getattr(caches[1], name))
    cache = caches[0]
    _same(*_both(monkeypatch, lambda: cache.gather(table, starts, 49)))
    _same(*_both(monkeypatch, lambda: cache.gather(table, starts, 49, dtype=dtype)))
    attention = PagedAttention.initialize(4, 2, 64, lookahead=1)
    cu = torch.tensor([0, 3, 4, 6] if ragged else [0, 2, 4, 6], dtype=I32, device=dev) if ragged else None
    q = fused[:6, :4]
    for kw in ({}, {"logsumexp": True}, {"window": 5}, {"scale": 0.3}, {"scale": 1}, {"output": torch.empty(6, 4, 64, dtype=dtype, device=dev)}):
        def call(kw=kw):
            found = attention(q, cache, table, tokens, cu_seqlens=cu, **kw)
            return found.clone() if torch.is_tensor(found) else found

        _same(*_both(monkeypatch, call))
    assert cache.device_error() == attention.device_error() == 0


def test_errors_are_the_same(dev, monkeypatch):
    from sonic_sampler_b200.interface import PagedAttention, ResidualNorm

    gen = torch.Generator().manual_seed(1)
    table, pages = ref.page_table([40, 2], 16, dev, gen)
    cache = ref.make_cache(pages, 16, 2, 64, BF16, dev, gen)
    tokens = torch.tensor([40, 2], dtype=I32, device=dev)
    x = torch.randn(2, 2, 64, device=dev).to(BF16)
    attention = PagedAttention.initialize(4, 2, 64)
    norm = ResidualNorm(torch.ones(64, dtype=BF16, device=dev))
    q = torch.randn(2, 4, 64, device=dev).to(BF16)
    wide = ResidualNorm(torch.ones(40000, dtype=BF16, device=dev))
    calls = [
        lambda: cache.append(x, x[:1], table, tokens), lambda: cache.append(x.float(), x.float(), table, tokens),
        lambda: cache.append(x.half(), x.half(), table, tokens), lambda: cache.append(x.cpu(), x.cpu(), table, tokens),
        lambda: cache.append(x[:1], x[:1], table, tokens), lambda: cache.append(x, x, table.long(), tokens),
        lambda: cache.append(x, x, table, tokens[:1]), lambda: cache.append(x, x, table, tokens, tokens),
        lambda: cache.append(x[..., 1:], x[..., 1:], table, tokens),
        lambda: cache.gather(table, tokens, 5), lambda: cache.gather(table, tokens.cpu(), 5), lambda: cache.gather(table, tokens, 5, dtype=F32),
        lambda: attention(q.half(), cache, table, tokens), lambda: attention(q[:, :3], cache, table, tokens),
        lambda: attention(q, cache, table, tokens, window=0), lambda: attention(q, cache, table, tokens, scale=math.inf),
        lambda: attention(q.cpu(), cache, table, tokens), lambda: attention(q, cache, table, tokens.cpu()),
        lambda: norm(x[0].float()), lambda: norm(x[0], x[0, :1]), lambda: norm(x[0].cpu()), lambda: norm(x[0, :, :63]),
        lambda: wide(torch.ones(1, 40000, dtype=BF16, device=dev)),
    ]
    for call in calls:
        def message(call=call):
            with pytest.raises((ValueError, RuntimeError)) as caught:
                call()
            return type(caught.value), str(caught.value)

        compiled, built = _both(monkeypatch, message)
        assert compiled == built


def test_nothing_is_kept(dev):
    """Outputs are freed with their last reference, and the arguments are not held."""
    from sonic_sampler_b200.interface import PagedAttention, ResidualNorm

    gen = torch.Generator().manual_seed(1)
    table, pages = ref.page_table([40, 2], 16, dev, gen)
    cache = ref.make_cache(pages, 16, 2, 64, E4M3, dev, gen, fill=0.0)
    tokens, starts = torch.tensor([40, 2], dtype=I32, device=dev), torch.tensor([0, 40, 42], dtype=I32, device=dev)
    x = torch.randn(2, 4, 64, device=dev).to(BF16)
    norm = ResidualNorm(torch.ones(64, dtype=BF16, device=dev), dtype=E4M3, group=128)
    attention = PagedAttention.initialize(4, 2, 64)

    def step():
        cache.append(x[:, :2], x[:, 2:], table, tokens)
        cache.gather(table, starts, 42)
        attention(x, cache, table, tokens)
        attention(x, cache, table, tokens, logsumexp=True)
        norm(x[0], x[1])
        norm(x[0])

    step()
    gc.collect()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(50):
        step()
    gc.collect()
    assert torch.cuda.memory_allocated() == held


def test_other_streams_and_graphs_use_the_current_stream(dev):
    from sonic_sampler_b200.interface import ResidualNorm

    x = torch.randn(64, 512, device=dev).to(BF16)
    norm = ResidualNorm(torch.ones(512, dtype=BF16, device=dev), dtype=E4M3)
    want = norm(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = norm(x)
    for t in got[:2]:
        t.view(torch.uint8).zero_()
    graph.replay()
    torch.cuda.synchronize()
    _same(got, want)


def test_the_module_refuses_wrong_argument_counts(dev):
    from sonic_sampler_b200 import _abi

    calls = _abi.load_calls()
    for function in (calls.norm, calls.append, calls.gather, calls.attention, calls.bind):
        with pytest.raises(TypeError, match="arguments"):
            function()
