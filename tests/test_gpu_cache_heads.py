"""The cache kernels with more kv heads than one CTA takes at once, and tokens of one and of many."""

from __future__ import annotations

import pytest
import torch

import decode_reference as ref
from test_gpu_cache import BF16, E4M3, F16, dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, E4M3)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("heads", [7, 32, 130])
@pytest.mark.parametrize("lengths", [[1], [40, 3, 0, 19]])
def test_many_heads(dev, dtype, cache_dtype, dim, heads, lengths):  # noqa: F811
    """Written rows, read back: a 16-bit cache gives them unchanged, an e4m3 one their codes times their
    scales rounded once."""
    gen = torch.Generator().manual_seed(heads)
    table, pages = ref.page_table(lengths, 16, dev, gen)
    cache = ref.make_cache(pages, 16, heads, dim, cache_dtype, dev, gen)
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
    total = sum(lengths)
    keys, values = ((torch.randn(total, heads, dim, generator=gen) * 3).to(dtype).to(dev) for _ in range(2))
    cache.append(keys, values, table, torch.tensor(lengths, dtype=torch.int32, device=dev), starts)
    got = cache.gather(table, starts, total, dtype=dtype)
    assert cache.device_error() == 0
    for x, y in zip((keys, values), got):
        if cache_dtype != E4M3:
            assert torch.equal(x, y)
            continue
        codes, scales = ref.quantise(x.double())
        # a tie may fall either way in fp32: then one step of the code, else the type's rounding
        quotient = x.double() * 448.0 / x.double().abs().amax(-1, keepdim=True).clamp(min=ref.FLOOR)
        step = ref.e4m3_step(quotient)
        tie = ((quotient / step) % 1.0 - 0.5).abs() * step <= 2.0 ** -22 * quotient.abs()
        exact = codes * scales[..., None]
        room = exact.abs() * (ref.EPS[dtype] + 2.0 ** -22) + ref.TINY[dtype] + torch.where(tie, step * scales[..., None], 0.0)
        assert ((y.double() - exact).abs() <= room).all()
