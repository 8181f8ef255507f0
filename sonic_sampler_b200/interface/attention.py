"""`PagedAttention`: attention of a step's new tokens over a paged key-value cache.

No counterpart in the reference, whose scope begins at the logits. One token a request is a decode
step; `lookahead + 1` tokens a request, each seeing the keys up to its own, are the target model's
side of a speculative verification (`UnshardedFusedMultistep` then judges its logits).
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch import Tensor

from sonic_sampler_b200 import _abi, ops
from sonic_sampler_b200._abi import FLAG_PDL
from sonic_sampler_b200.core.cache import PagedCache
from sonic_sampler_b200.core.described import Described
from sonic_sampler_b200.interface.base import default_device


@dataclass(eq=False)
class PagedAttention(Described):
    q_heads: int
    kv_heads: int
    head_dim: int
    lookahead: int
    pdl: bool
    # zero-filled workspace of the kernel; calls that overlap on the GPU need objects of their own
    scratchpad: Tensor

    def describe(self) -> None:
        self.template = ops.paged_attention_template(self.q_heads, self.head_dim, FLAG_PDL if self.pdl else 0)
        self.address = ctypes.addressof(self.template)

    @classmethod
    def initialize(cls, q_heads: int, kv_heads: int, head_dim: int, lookahead: int = 0, pdl: bool = True) -> "PagedAttention":
        if q_heads < 1 or kv_heads < 1 or q_heads % kv_heads:
            raise ValueError(f"q_heads must be a multiple of kv_heads, got {q_heads} and {kv_heads}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if lookahead < 0:
            raise ValueError(f"lookahead must not be negative, got {lookahead}")
        if lookahead >= ops.INT32_MAX:
            raise ValueError(f"lookahead must be below 2^31 - 1, got {lookahead}")
        return cls(q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, lookahead=lookahead, pdl=pdl,
                   scratchpad=ops.new_workspace(ops.paged_attention_workspace_bytes(), default_device()))

    def device_error(self) -> int:
        """Read and clear the device error word: 0, or DEVICE_ERR_PAGE when a call met a page id
        outside the cache or a length outside its page-table row (that request's output is then
        unspecified). Synchronises the current stream."""
        return ops.workspace_error(self.scratchpad)

    def __call__(self, queries: Tensor, cache: PagedCache, page_table: Tensor, lengths: Tensor,
                 cu_seqlens: Tensor | None = None, window: int | None = None, scale: float | None = None,
                 logsumexp: bool = False, output: Tensor | None = None) -> Tensor | tuple[Tensor, Tensor]:
        """Attention of `queries` `[tokens, q_heads, head_dim]` (bf16 or fp16; the cache's dtype
        unless it is e4m3) over the cached tokens of their requests, their own included.

        Rows `cu_seqlens[b]:cu_seqlens[b + 1]` (without it, tokens / requests rows each) are the
        last tokens of request b, which has `lengths[b]` in the cache. Each sees the keys up to its
        own position, the last `window` of them where that is given. `scale` is 1 / sqrt(head_dim)
        by default. `lookahead` of `initialize` is a hint: requests may bring more tokens with
        `cu_seqlens`, but slowly (give prompts an object of their own).

        Returns the output (in `output` where that is given), and with `logsumexp` also the fp32
        `[tokens, q_heads]` logarithms of the softmax sums, with which outputs over disjoint key
        ranges can be joined. A query that sees no key gives zeros and -infinity, and so do rows outside
        every request (a padded call's, before `cu_seqlens[0]` or from `cu_seqlens[-1]` on)."""
        struct, device, scratchpad = cache.struct, cache.device, self.scratchpad
        if struct.kv_heads != self.kv_heads or struct.head_dim != self.head_dim:
            raise ValueError("the cache's kv_heads and head_dim must match `initialize`'s")
        if output is None and scratchpad.device == device:
            found = _abi.load_calls().attention(self.address, cache.address, device.index, scratchpad.data_ptr(), scratchpad.numel(),
                                                queries, page_table, lengths, cu_seqlens, self.lookahead + 1, window, scale,
                                                logsumexp)
            if found is not None and type(found) is not int:
                return found
        ops._require_cuda(queries)
        if window is None:
            window = 0
        elif window < 1:
            raise ValueError(f"`window` must be positive, got {window}")
        if scratchpad.device != device:
            raise ValueError(f"the cache is on {device}, this object's workspace on {scratchpad.device}")
        args, out, lse = ops.paged_attention_args(
            self.template, struct, queries, page_table, lengths, cu_seqlens=cu_seqlens,
            max_tokens=self.lookahead + 1 if cu_seqlens is not None else 0, window=window, scale=scale, out=output,
            logsumexp=logsumexp, workspace=scratchpad, device=device)
        ops.launch_paged_attention(args, device)
        return (out, lse) if logsumexp else out
