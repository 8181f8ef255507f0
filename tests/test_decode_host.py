"""Host side of the decode-side operators, without a GPU: struct layouts, argument checks before any
CUDA call, and no CPU fallback."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from sonic_sampler_b200 import _abi, ops

HEADER = Path(__file__).resolve().parents[1] / "include" / "sonic_b200.h"
BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn
FAKE = 1 << 20  # an aligned address that no check dereferences


@pytest.fixture(scope="module")
def lib():
    from sonic_sampler_b200 import build

    build.build()
    return _abi.load_library()


def _status(lib, fn, args):
    return getattr(lib, fn)(ctypes.byref(args), None), lib.sonic_last_error().decode()


def test_struct_layout_matches_header():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for cname, pyt in (("SonicPagedCache", _abi.PagedCacheStruct), ("SonicSequences", _abi.SequencesStruct),
                       ("SonicCacheAppendArgs", _abi.CacheAppendArgs), ("SonicCacheGatherArgs", _abi.CacheGatherArgs),
                       ("SonicPagedAttentionArgs", _abi.PagedAttentionArgs), ("SonicResidualNormArgs", _abi.ResidualNormArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, flags=re.S).group(1)
        fields = [re.findall(r"(\w+)\s*$", d.strip())[0] for d in body.split(";") if d.strip()]
        assert fields == [f for f, _ in pyt._fields_], cname


def _cache(a):
    c = a.cache
    c.keys = c.values = FAKE
    c.dtype, c.pages, c.page_size, c.kv_heads, c.head_dim = _abi.DT_BF16, 4, 16, 2, 64
    c.page_stride, c.head_stride, c.slot_stride = 2048, 1024, 64
    s = a.sequences
    s.requests, s.tokens, s.page_table, s.table_stride, s.table_width, s.lengths = 2, 4, FAKE, 3, 3, FAKE
    return a


def _append():
    a = _cache(_abi.CacheAppendArgs())
    a.dtype, a.keys, a.values = _abi.DT_BF16, FAKE, FAKE
    a.key_token_stride = a.value_token_stride = 128
    a.key_head_stride = a.value_head_stride = 64
    return a


def _gather():
    a = _cache(_abi.CacheGatherArgs())
    a.dtype, a.starts, a.keys, a.values = _abi.DT_BF16, FAKE, FAKE, FAKE
    return a


def _attention():
    a = _cache(_abi.PagedAttentionArgs())
    a.dtype, a.q_heads, a.scale = _abi.DT_BF16, 4, 0.125
    a.queries, a.out, a.workspace, a.workspace_bytes = FAKE, FAKE, FAKE, 1 << 30
    a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride = 256, 64, 256, 64
    return a


def _set(a, path, value):
    *outer, last = path.split(".")
    for name in outer:
        a = getattr(a, name)
    setattr(a, last, value)


CACHE_CHECKS = [
    ("cache.keys", None, "cache keys"), ("cache.values", None, "cache keys"), ("cache.dtype", _abi.DT_F32, "cache dtype"),
    ("cache.head_dim", 96, "head_dim"), ("cache.pages", 0, "positive"), ("cache.page_size", 0, "positive"),
    ("cache.kv_heads", 0, "positive"), ("cache.kv_heads", 2000, "kv_heads"), ("cache.keys", FAKE + 8, "16-byte"),
    ("cache.slot_stride", 68, "16-byte"), ("cache.head_stride", -64, "negative"), ("cache.dtype", _abi.DT_E4M3, "scales"),
    ("sequences.requests", 0, "requests"), ("sequences.tokens", -1, "tokens"), ("sequences.page_table", None, "page_table"),
    ("sequences.table_width", 0, "page_table"), ("sequences.table_stride", -1, "page_table"),
]
TOKEN_CHECKS = [("sequences.lengths", None, "lengths"), ("sequences.tokens", 3, "multiple of requests")]
OWN_CHECKS = {
    "sonic_cache_append": (_append, TOKEN_CHECKS + [
        ("dtype", _abi.DT_F32, "bf16 or f16"), ("dtype", _abi.DT_F16, "cache's dtype"), ("keys", None, "NULL"),
        ("values", FAKE + 2, "16-byte"), ("key_token_stride", 129, "16-byte"), ("value_head_stride", 4, "16-byte")]),
    "sonic_cache_gather": (_gather, [
        ("dtype", _abi.DT_F32, "bf16 or f16"), ("dtype", _abi.DT_F16, "cache's dtype"), ("starts", None, "NULL"),
        ("keys", None, "NULL"), ("values", FAKE + 4, "16-byte")]),
    "sonic_paged_attention": (_attention, TOKEN_CHECKS + [
        ("dtype", _abi.DT_F32, "bf16 or f16"), ("dtype", _abi.DT_F16, "cache's dtype"), ("q_heads", 3, "multiple of kv_heads"),
        ("q_heads", 0, "multiple of kv_heads"), ("window", -1, "window"), ("max_tokens", -1, "max_tokens"),
        ("scale", math.nan, "finite"), ("scale", math.inf, "finite"), ("queries", None, "NULL"), ("out", None, "NULL"),
        ("queries", FAKE + 8, "16-byte"), ("q_head_stride", 68, "16-byte"), ("out", FAKE + 4, "8-byte"),
        ("out_token_stride", 258, "8-byte"), ("workspace", None, "workspace"), ("workspace_bytes", 100, "workspace"),
        ("workspace", FAKE + 8, "workspace"), ("sequences.tokens", 2 ** 31 - 2, "too large"),
        ("sequences.table_width", 2 ** 31 - 1, "2\\^32 steps")]),
}


@pytest.mark.parametrize("entry", list(OWN_CHECKS))
def test_entries_refuse_on_the_host(lib, entry):
    make, own = OWN_CHECKS[entry]
    assert getattr(lib, entry)(None, None) == _abi.SONIC_ERR_INVALID_ARGUMENT
    for path, value, message in CACHE_CHECKS + own:
        a = make()
        _set(a, path, value)
        if path == "sequences.table_width" and value > 100:
            a.sequences.requests, a.sequences.tokens = 1 << 10, 1 << 10
        status, text = _status(lib, entry, a)
        assert status in (_abi.SONIC_ERR_INVALID_ARGUMENT, _abi.SONIC_ERR_UNSUPPORTED, _abi.SONIC_ERR_WORKSPACE), path
        assert re.search(message, text), (path, value, text)
    a = make()
    a.sequences.tokens = 0
    assert _status(lib, entry, a)[0] == _abi.SONIC_OK  # nothing to do, nothing launched


def test_norm_refuses_on_the_host(lib):
    def make():
        a = _abi.ResidualNormArgs()
        a.rows, a.hidden, a.dtype, a.out_dtype = 2, 64, _abi.DT_BF16, _abi.DT_BF16
        a.x = a.weight = a.out = FAKE
        return a

    for path, value, message in (
            ("rows", -1, "rows"), ("hidden", 0, "hidden"), ("hidden", 40000, "32768"), ("dtype", _abi.DT_E4M3, "dtype"),
            ("out_dtype", _abi.DT_F32, "out_dtype"), ("group", 128, "group"), ("x", None, "NULL"), ("weight", None, "NULL"),
            ("out", None, "NULL"), ("out_dtype", _abi.DT_E4M3, "scales")):
        a = make()
        _set(a, path, value)
        status, text = _status(lib, "sonic_residual_norm", a)
        assert status in (_abi.SONIC_ERR_INVALID_ARGUMENT, _abi.SONIC_ERR_UNSUPPORTED) and message in text, (path, text)
    a = make()
    a.out_dtype, a.group, a.scales = _abi.DT_E4M3, 64, FAKE
    assert "group" in _status(lib, "sonic_residual_norm", a)[1]
    a = make()
    a.rows = 0
    assert _status(lib, "sonic_residual_norm", a)[0] == _abi.SONIC_OK


def test_workspace_query(lib):
    assert lib.sonic_paged_attention_workspace_size(None) == 0
    assert ops.paged_attention_workspace_bytes() > 1 << 20


def test_no_cpu_fallback():
    from sonic_sampler_b200.interface import PagedAttention, PagedCache, ResidualNorm

    cache = PagedCache.allocate(3, 16, 2, 64, device="cpu")
    assert cache.page_size == 16 and cache.keys.shape == (3, 2, 16, 64)
    x = torch.zeros(2, 2, 64, dtype=BF16)
    table, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        cache.append(x, x, table, lengths)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        cache.gather(table, torch.zeros(3, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        PagedAttention.initialize(4, 2, 64)(x.repeat(1, 2, 1), cache, table, lengths)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ResidualNorm(torch.ones(64, dtype=BF16))(x)


def test_an_e4m3_cache_brings_its_scales():
    from sonic_sampler_b200.interface import PagedCache

    cache = PagedCache.allocate(3, 16, 2, 64, dtype=E4M3, device="cpu")
    assert cache.key_scales.shape == (3, 2, 16) and cache.key_scales.dtype == torch.float32
    assert cache.struct.scale_page_stride == 32 and cache.struct.scale_head_stride == 16
    with pytest.raises(ValueError, match="key_scales"):
        PagedCache(cache.keys, cache.values, cache.key_scales[:2], cache.value_scales[:2])
    with pytest.raises(ValueError, match="bf16, fp16 or float8"):
        PagedCache(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))
