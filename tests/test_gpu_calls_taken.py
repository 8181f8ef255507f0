"""Which calls the compiled module takes: the usual forms come back from it, others it passes on to the
builders, which would otherwise make every call without anyone noticing."""

from __future__ import annotations

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


class Spy:
    """The compiled module, with what its functions gave."""

    def __init__(self, calls):
        self.calls, self.given = calls, []

    def __getattr__(self, name):
        def call(*args):
            self.given.append((name, getattr(self.calls, name)(*args)))
            return self.given[-1][1]

        return call


@pytest.fixture
def taken(monkeypatch):
    """taken(name, call) -> what the module's function `name` gave in `call()`, which calls it once."""
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    spy = Spy(_abi.load_calls())
    monkeypatch.setattr(_abi, "_CALLS", spy)

    def run(name, call):
        spy.given.clear()
        found = call()
        assert [n for n, _ in spy.given] == [name]
        given = spy.given[0][1]
        if isinstance(given, (tuple, torch.Tensor)):
            assert given is found
        return given

    return run


DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out,group", [(None, None), (E4M3, None), (E4M3, 128)])
def test_norm(taken, dtype, out, group):
    from sonic_sampler_b200.interface import ResidualNorm

    norm = ResidualNorm(torch.ones(200, dtype=dtype, device=DEV), dtype=out, group=group)
    x = torch.randn(5, 203, device=DEV).to(dtype)[:, :200]
    for args in ((x,), (x, x), (x[:0],), (torch.nn.Parameter(x), x)):
        given = taken("norm", lambda args=args: norm(*args))
        assert type(given) is tuple and len(given) == 3
        assert (given[1] is None) == (out is None) and (given[2] is None) == (len(args) == 1)
    assert taken("norm", lambda: norm(x[:, None].contiguous().view(5, 200))) is not None
    with pytest.raises(ValueError):
        assert taken("norm", lambda: norm(x[:, :199])) is None


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
def test_cache_and_attention(taken, dtype, cache_dtype):
    from sonic_sampler_b200.interface import PagedAttention

    dev, gen = torch.device(DEV), torch.Generator().manual_seed(1)
    lengths = [40, 2, 7]
    table, pages = ref.page_table(lengths, 16, dev, gen)
    tokens, starts = torch.tensor(lengths, dtype=I32, device=dev), torch.tensor([0, 40, 42, 49], dtype=I32, device=dev)
    cache = ref.make_cache(pages, 16, 2, 64, cache_dtype, dev, gen)
    fused = torch.randn(49, 8, 64, generator=gen).to(dtype).to(dev)
    assert taken("append", lambda: cache.append(fused[:, 4:6], fused[:, 6:], table, tokens, starts)) == 0
    assert taken("append", lambda: cache.append(fused[:3, 4:6], fused[:3, 6:], table, tokens)) == 0
    for kw in ({}, {"dtype": dtype}):
        if cache_dtype == E4M3 or kw:
            assert type(taken("gather", lambda kw=kw: cache.gather(table, starts, 49, **kw))) is tuple
    attention = PagedAttention.initialize(4, 2, 64, lookahead=1)
    cu = torch.tensor([0, 3, 4, 6], dtype=I32, device=dev)
    q = fused[:6, :4]
    for kw in ({}, {"cu_seqlens": cu}, {"window": 5}, {"scale": 0.3}, {"cu_seqlens": cu, "window": 3, "scale": 0.25}):
        assert torch.is_tensor(taken("attention", lambda kw=kw: attention(q, cache, table, tokens, **kw)))
        given = taken("attention", lambda kw=kw: attention(q, cache, table, tokens, logsumexp=True, **kw))
        assert type(given) is tuple and len(given) == 2
    # other forms: passed on
    assert taken("attention", lambda: attention(q, cache, table, tokens, scale=1)) is None
    with pytest.raises(ValueError):
        taken("attention", lambda: attention(q, cache, table, tokens, window=0))
    with pytest.raises(ValueError):
        taken("append", lambda: cache.append(q[:, :1], q[:, :1], table, tokens))
