"""The type that a read-back has where one of its outputs is given."""

from __future__ import annotations

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("given", ["keys", "values", "both"])
def test_one_given_output_says_the_type(dtype, given):
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    dev, gen = torch.device("cuda:0"), torch.Generator().manual_seed(1)
    table, pages = ref.page_table([40, 2], 16, dev, gen)
    cache = ref.make_cache(pages, 16, 2, 64, E4M3, dev, gen)
    ref.fill_cache(cache, table, [40, 2], gen)
    starts = torch.tensor([0, 40, 42], dtype=torch.int32, device=dev)
    want = cache.gather(table, starts, 42, dtype=dtype)
    room = {name: torch.empty(42, 2, 64, dtype=dtype, device=dev) for name in ("keys", "values") if given in (name, "both")}
    found = cache.gather(table, starts, 42, **room)
    for name, got, expect in zip(("keys", "values"), found, want):
        assert got is room.get(name, got) and got.dtype == dtype and torch.equal(got, expect)
