"""Fields of the decode-side objects assigned after their construction: what the calls use follows them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from sonic_sampler_b200 import _abi
from sonic_sampler_b200.interface import PagedAttention, PagedCache, ResidualNorm

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def test_cache_follows_its_tensors():
    cache = PagedCache.allocate(3, 16, 2, 64, dtype=E4M3, device="cpu")
    errors = cache.errors
    keys, scales = torch.zeros(3, 2, 16, 64, dtype=E4M3), torch.ones(3, 2, 16)
    cache.keys = keys
    cache.value_scales = scales
    assert cache.struct.keys == keys.data_ptr() and cache.struct.value_scales == scales.data_ptr()
    assert cache.address == cache.place[0] == ctypes.addressof(cache.struct)
    assert cache.errors is errors and cache.place[3] == errors.data_ptr()
    cache.pdl = False
    assert cache.flags == cache.place[2] == 0
    cache.pdl = True
    assert cache.flags == cache.place[2] == _abi.FLAG_PDL


def test_cache_refuses_a_tensor_that_does_not_fit_and_keeps_its_own():
    cache = PagedCache.allocate(3, 16, 2, 64, device="cpu")
    keys, values, struct = cache.keys, cache.values, cache.struct
    for name, t in (("keys", keys[:2]), ("values", values.half()), ("keys", keys.transpose(1, 2).contiguous().transpose(1, 2)),
                    ("key_scales", torch.ones(3, 2, 16))):
        with pytest.raises(ValueError):
            setattr(cache, name, t)
        assert cache.keys is keys and cache.values is values and cache.key_scales is None and cache.struct is struct


def test_norm_follows_its_fields():
    norm = ResidualNorm(torch.ones(64, dtype=BF16), eps=1e-5)
    norm.eps = 0.5
    assert norm.template.eps == 0.5 and norm.address == ctypes.addressof(norm.template)
    norm.dtype = E4M3
    norm.group = 128
    norm.pdl = False
    assert (norm.template.out_dtype, norm.template.group, norm.template.flags) == (_abi.DT_E4M3, 128, 0)
    norm.weight = torch.ones(96, dtype=F16)
    assert (norm.template.hidden, norm.template.dtype) == (96, _abi.DT_F16)
    assert norm.address == ctypes.addressof(norm.template)
    for name, bad in (("eps", -1.0), ("group", 64), ("dtype", torch.float32), ("weight", torch.ones(64, 2, dtype=BF16)[:, 0])):
        old = getattr(norm, name)
        with pytest.raises(ValueError):
            setattr(norm, name, bad)
        assert getattr(norm, name) is old


def test_attention_follows_its_fields():
    attention = PagedAttention.initialize(4, 2, 64)
    attention.q_heads = 8
    attention.pdl = False
    attention.head_dim = 256
    assert (attention.template.q_heads, attention.template.flags, attention.template.scale) == (8, 0, 0.0625)
    assert attention.address == ctypes.addressof(attention.template)
