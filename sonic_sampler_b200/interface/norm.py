"""`ResidualNorm`: root-mean-square norm with the residual's addition and an output in 8 bits.

No counterpart in the reference: it is the step between a served model's layers, and before the
projection whose logits the sampler reads.
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
class ResidualNorm(Described):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight, in fp32.

    `dtype=torch.float8_e4m3fn` returns y's e4m3 codes, with an fp32 scale per row or per `group`
    (128) columns: y stands for code * scale. Otherwise y is rounded to the input's dtype."""

    weight: Tensor
    eps: float = 1e-6
    dtype: torch.dtype | None = None
    group: int | None = None
    pdl: bool = True

    def describe(self) -> None:
        if self.dtype not in (None, E4M3, self.weight.dtype):
            raise ValueError(f"`dtype` must be float8_e4m3fn or the weight's {self.weight.dtype}, got {self.dtype}")
        if self.group not in (None, 128) or (self.group and self.dtype != E4M3):
            raise ValueError(f"`group` must be 128 (with a float8_e4m3fn output) or None, got {self.group}")
        if not self.eps >= 0.0:
            raise ValueError(f"`eps` must not be negative, got {self.eps}")
        self.template = ops.residual_norm_template(self.weight, self.dtype, self.eps, self.group or 0, FLAG_PDL if self.pdl else 0)
        self.address = ctypes.addressof(self.template)

    def __call__(self, x: Tensor, residual: Tensor | None = None, residual_out: Tensor | None = None, out: Tensor | None = None,
                 scales: Tensor | None = None) -> tuple[Tensor, Tensor | None, Tensor | None]:
        """(y, scales, r) of rows `x` `[..., hidden]`, in the weight's dtype (bf16, fp16 or fp32).

        `scales` is None unless the output is in 8 bits (`[..., 1]` or `[..., ceil(hidden / 128)]`);
        r, rounded to the input's dtype, is None without a `residual`. `out`, `scales` and
        `residual_out` may give the tensors to write; `residual_out` may be `residual` or `x`."""
        if residual_out is None and out is None and scales is None:
            found = _abi.load_calls().norm(self.address, x, self.weight, residual)
            if type(found) is tuple:
                return found
        ops._require_cuda(x)
        if x.dim() != 2:
            def rows(t):
                return t if t is None else t.view(-1, t.size(-1))

            y, scales, r = self(rows(x), rows(residual), rows(residual_out), rows(out), rows(scales))
            lead = x.shape[:-1]
            return tuple(t if t is None else t.view(*lead, t.size(-1)) for t in (y, scales, r))
        args, out, scales, residual_out = ops.residual_norm_args(self.template, x, self.weight, residual, residual_out, out, scales)
        ops.launch_residual_norm(args, x.device)
        return out, scales, residual_out
