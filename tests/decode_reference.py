"""64-bit restatements of the decode-side operators, and inputs for their tests.

Attention is restated per query over the keys it sees and nothing else, so that what lies at unseen
positions (unwritten slots, other requests' pages, NaN) cannot reach it. Each restatement returns
with its values a bound on the error that the arithmetic of the kernels may have: fp32 sums, one
rounding of each softmax weight and one of the result."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
FLOOR = 2.0 ** -60
#: relative rounding error (half a step) of a value of each type
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
#: half the smallest step of fp16; the other types' is far below any tolerance here
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def e4m3(v):
    """Nearest e4m3 value of fp64 values, ties to even, saturated; NaN stays."""
    exponent = torch.frexp(v).exponent.double() - 1.0
    step = torch.exp2(exponent.clamp(min=-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def e4m3_step(v):
    """Distance of neighbouring e4m3 values around v."""
    exponent = torch.frexp(v).exponent.double() - 1.0
    return torch.exp2(exponent.clamp(min=-6.0) - 3.0)


def quantise(x):
    """(codes as fp64 values, scales) of the rows of fp64 x."""
    c = x.abs().amax(-1, keepdim=True).clamp(min=FLOOR)
    return e4m3(x * 448.0 / c), (c / 448.0).squeeze(-1)


def make_cache(pages, page_size, kv_heads, head_dim, dtype, device, gen, fill=math.nan, layout="heads"):
    """An empty cache whose every slot holds `fill` (NaN codes and scales in 8 bits).

    layout "slots" lays a page out as [slot, head, dim], "padded" leaves a gap after every row."""
    from sonic_sampler_b200.interface import PagedCache

    def pages_of():
        if layout == "slots":
            t = torch.empty(pages, page_size, kv_heads, head_dim, dtype=dtype, device=device).transpose(1, 2)
        elif layout == "padded":
            t = torch.empty(pages, kv_heads, page_size, head_dim + 16, dtype=dtype, device=device)[..., :head_dim]
        else:
            t = torch.empty(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        t.view(torch.uint8).fill_(0x7f) if dtype == E4M3 else t.fill_(fill)
        return t

    scales = [torch.full((pages, kv_heads, page_size), fill, device=device) if dtype == E4M3 else None for _ in range(2)]
    return PagedCache(pages_of(), pages_of(), *scales)


def page_table(lengths, page_size, device, gen, spare=2, extra=1):
    """Distinct random pages for every request; unused entries hold an id outside any cache."""
    counts = [-(-n // page_size) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lengths), max(counts + [0]) + extra), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.to(device), pages


def fill_cache(cache, table, lengths, gen, scale=1.0):
    """Write random tokens into every live position of the cache with plain torch operations;
    returns the (keys, values) that the cache stands for, per request [length, heads, dim] in fp64."""
    _, heads, size, dim = cache.keys.shape
    held = []
    for b, n in enumerate(lengths):
        position = torch.arange(n, device=cache.device)
        page, slot = table[b].long()[position // size], position % size
        pair = []
        for data, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
            x = torch.randn(n, heads, dim, generator=gen, dtype=torch.float64).to(cache.device) * scale
            x *= torch.exp(torch.randn(n, heads, 1, generator=gen, dtype=torch.float64)).to(cache.device)
            if scales is None:
                x = x.to(data.dtype)
                data[page, :, slot] = x
                x = x.double()
            elif n:
                codes, s = quantise(x.float().double())
                codes, s = codes.to(torch.float32).to(E4M3), s.float()
                data.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
                scales[page, :, slot] = s
                x = codes.double() * s.double()[..., None]
            pair.append(x)
        held.append(tuple(pair))
    return held


def attention(q, held, lengths, new, first, kv_heads, window=None, scale=None, weight_eps=None, out_dtype=None):
    """(out, out bound, lse, lse bound) of queries q [tokens, q_heads, dim] over `held`."""
    tokens, heads, dim = q.shape
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device=q.device)
    out_bound = torch.full_like(out, 1e-30)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.full_like(lse, 1e-30)
    for b, length in enumerate(lengths):
        keys, values = held[b]
        for i in range(new[b]):
            last = length - new[b] + i
            start = max(0, last - window + 1) if window else 0
            if last < start:
                continue
            row = q[first[b] + i].double().view(kv_heads, group, dim)
            k, v = keys[start:last + 1].transpose(0, 1), values[start:last + 1].transpose(0, 1)  # [heads, keys, dim]
            s = torch.einsum("hgd,hkd->hgk", row, k) * scale
            total = torch.logsumexp(s, -1)
            p = torch.exp(s - total[..., None])
            spread = torch.einsum("hgk,hkd->hgd", p, v.abs())
            # fp32 products summed in any order (tensor cores may truncate: 4 units instead of a half),
            # and the rounding of the score itself on its way into the exponential
            terms = torch.einsum("hgd,hkd->hgk", row.abs(), k.abs()).amax(-1) * scale
            delta = 2.0 ** -22 * ((dim + 8) * terms + 8)
            n = k.size(1)
            at = first[b] + i
            out[at] = torch.einsum("hgk,hkd->hgd", p, v).reshape(heads, dim)
            lse[at] = total.reshape(heads)
            sums = 2.0 ** -22 * (n + 64)
            out_bound[at] = (spread * (2 * delta[..., None] + sums + 1.01 * weight_eps)
                             + out[at].view(kv_heads, group, dim).abs() * 1.01 * EPS[out_dtype] + TINY[out_dtype]).reshape(heads, dim)
            lse_bound[at] = (delta + sums + 2.0 ** -22 * total.abs()).reshape(heads)
    return out, out_bound, lse, lse_bound


def norm(x, residual, weight, eps):
    r = x.double() if residual is None else x.double() + residual.double()
    return r, r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * weight.double()
