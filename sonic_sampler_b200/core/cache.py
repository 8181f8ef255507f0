"""`PagedCache`: the keys and values of one layer in pages, written and read back by batched calls.

No counterpart in the reference, whose scope is the sampler: this is the cache that the served
model's attention (`interface/attention.py`) reads between two sampler calls.

A request's token at position t lies in page `page_table[b, t // page_size]`, slot
`t % page_size`. `lengths[b]` counts the request's tokens in the cache, those of the call included,
so after a verification the next step's lengths are `lengths + offsets + 1`: what a rejected draft
wrote lies past the new length and is overwritten by the next tokens.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch import Tensor

from sonic_sampler_b200 import _abi, ops
from sonic_sampler_b200._abi import FLAG_PDL
from sonic_sampler_b200.core.described import Described

E4M3 = torch.float8_e4m3fn


@dataclass(eq=False)
class PagedCache(Described):
    """Pages of keys and values, `[pages, kv_heads, page_size, head_dim]` in bf16, fp16 or
    float8_e4m3fn; with float8_e4m3fn one fp32 scale per (page, head, slot), and a row stands for
    code * scale. Any strides with a unit inner one, shared by keys and values, rows on 16-byte
    boundaries. The calls after an assignment to a field use the new tensor, which must fit the others:
    pages of another form make another PagedCache."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor | None = None
    value_scales: Tensor | None = None
    pdl: bool = True

    def describe(self) -> None:
        struct = ops.paged_cache_struct(self.keys, self.values, self.key_scales, self.value_scales)
        device = self.keys.device
        # the device error word of append and gather
        errors = getattr(self, "errors", None)
        self.errors = errors if errors is not None and errors.device == device else ops.new_workspace(256, device)
        self.struct, self.device = struct, device
        self.flags = FLAG_PDL if self.pdl else 0
        # what `_abi.load_calls()`'s functions take of it
        self.address = ctypes.addressof(struct)
        self.place = (self.address, device.index, self.flags, self.errors.data_ptr())

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str | None = None, pdl: bool = True) -> "PagedCache":
        """A cache whose pages hold no tokens yet (zeros)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        keys, values = (torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        scales = [torch.zeros(pages, kv_heads, page_size, device=device) if dtype == E4M3 else None for _ in range(2)]
        return cls(keys, values, *scales, pdl=pdl)

    @property
    def page_size(self) -> int:
        return self.keys.size(2)

    def append(self, keys: Tensor, values: Tensor, page_table: Tensor, lengths: Tensor,
               cu_seqlens: Tensor | None = None) -> "PagedCache":
        """Write the call's new tokens, `[tokens, kv_heads, head_dim]` in bf16 or fp16 (the cache's
        own dtype unless it is e4m3; any token and head strides, rows on 16-byte boundaries).

        Request b's are its last n_b positions: rows `cu_seqlens[b]:cu_seqlens[b + 1]`, or without
        `cu_seqlens` tokens / requests rows each. An e4m3 row gets the scale c / 448, c the larger of
        its largest magnitude and 2^-60, and its codes are rounded to nearest even. Runs on the
        current stream; a token whose page is not in the cache is skipped and recorded
        (`device_error`)."""
        status = _abi.load_calls().append(*self.place, keys, values, page_table, lengths, cu_seqlens)
        if status == 0:
            return self
        ops._require_cuda(keys)
        args = ops.cache_append_args(self.struct, keys, values, page_table, lengths, cu_seqlens=cu_seqlens,
                                     flags=self.flags, error=self.errors, device=self.device)
        ops.launch_cache_append(args, self.device)
        return self

    def gather(self, page_table: Tensor, starts: Tensor, total: int, dtype: torch.dtype | None = None,
               keys: Tensor | None = None, values: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """Read back positions `[0, starts[b + 1] - starts[b])` of every request as contiguous
        `[total, kv_heads, head_dim]` keys and values, request b's from row `starts[b]` on
        (`total` is the host's copy of `starts[-1]`).

        An e4m3 row is code * scale, rounded once to `dtype` (bf16 by default, or fp16); other caches
        keep their dtype. `keys` and `values` may give the outputs to write."""
        if dtype is None:
            given = values if keys is None else keys
            dtype = given.dtype if given is not None else torch.bfloat16 if self.keys.dtype == E4M3 else self.keys.dtype
        if keys is None and values is None and (dtype == torch.bfloat16 or dtype == torch.float16):
            rows = _abi.load_calls().gather(*self.place, page_table, starts, total, dtype == torch.float16)
            if type(rows) is tuple:
                return rows
        ops._require_cuda(page_table)
        args, keys, values = ops.cache_gather_args(self.struct, page_table, starts, total, dtype, keys, values, flags=self.flags,
                                                   error=self.errors, device=self.device)
        ops.launch_cache_gather(args, self.device)
        return keys, values

    def device_error(self) -> int:
        """Read and clear the error word of earlier `append` and `gather` calls: 0, or
        DEVICE_ERR_PAGE when a token's page was not in the cache. Synchronises the current stream."""
        return ops.workspace_error(self.errors)
