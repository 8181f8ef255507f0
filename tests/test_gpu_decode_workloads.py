"""The decode-side workloads run, and what they are run on is as described."""

import pytest
import torch

from sonic_sampler_b200 import workloads


def test_paged_tokens_hand_out_every_page_once():
    table, lengths, pages = workloads.paged_tokens([1, 16, 17, 50], 16, "cpu", 0)
    assert pages == 8 and table.shape == (4, 4) and lengths.tolist() == [1, 16, 17, 50]
    used = [p for row, n in zip(table.tolist(), (1, 1, 2, 4)) for p in row[:n]]
    assert sorted(used) == list(range(8))


@pytest.mark.gpu
@pytest.mark.parametrize("name", workloads.DECODE_SIDE)
def test_decode_side_workloads(name):
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    found = workloads.runner(name, "cuda")()
    for t in found if isinstance(found, tuple) else (found,):
        if torch.is_tensor(t):
            assert torch.isfinite(t.float()).all()
    if name.startswith("cache_append"):
        assert found.device_error() == 0
