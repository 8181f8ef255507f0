"""A small decoder served end to end: residual norm, paged cache, attention over it, sampler.

    python -m sonic_sampler_b200.decode [--requests 8] [--prompt 200] [--steps 32] [--lookahead 3]
                                        [--cache e4m3|bf16]

No counterpart in the reference, whose scope begins at the logits. The weights are random and
positions are not encoded: it shows how the operators are called between two sampler calls, and the
tests hold their composition against itself. Projections are plain library products, in 8 bits
after a norm with an 8-bit output.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import Tensor

from sonic_sampler_b200 import workloads
from sonic_sampler_b200.interface import (
    PagedAttention,
    PagedCache,
    ResidualNorm,
    UnshardedFusedMultistep,
    UnshardedFusedSingular,
)

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn
I32 = torch.int32


class Projection:
    """x @ weight for the output of a norm: bf16, or e4m3 codes with a scale per row (the weight is
    then held in e4m3 with a scale per column)."""

    def __init__(self, weight: Tensor, eight_bits: bool):
        self.weight, self.scales = weight, None
        if eight_bits:
            self.scales = weight.float().abs().amax(0, keepdim=True) / 448.0
            # _scaled_mm reads its second operand column by column
            self.weight = (weight.float() / self.scales).to(E4M3).t().contiguous().t()

    def __call__(self, x: Tensor, scales: Tensor | None) -> Tensor:
        if self.scales is None:
            return x @ self.weight
        return torch._scaled_mm(x, self.weight, scale_a=scales, scale_b=self.scales, out_dtype=BF16)


@dataclass
class Layer:
    norm: ResidualNorm
    qkv: Projection
    out: Tensor
    mlp_norm: ResidualNorm
    up: Projection
    down: Tensor
    cache: PagedCache


class Decoder:
    """`layers` of attention and gated MLP over `hidden` columns. One attention object serves every
    layer: its calls follow one another on the stream."""

    def __init__(self, vocab: int = 32000, hidden: int = 512, layers: int = 2, q_heads: int = 8, kv_heads: int = 2,
                 head_dim: int = 64, pages: int = 1024, page_size: int = 16, lookahead: int = 0, cache: torch.dtype = BF16,
                 eight_bits: bool = False, seed: int = 0, device: torch.device | str = "cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows: int, columns: int) -> Tensor:
            return (torch.randn(rows, columns, generator=g, device=device) * rows**-0.5).to(BF16)

        def norm(dtype: torch.dtype | None) -> ResidualNorm:
            return ResidualNorm((1.0 + 0.1 * torch.randn(hidden, generator=g, device=device)).to(BF16), dtype=dtype)

        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.embedding = torch.randn(vocab, hidden, generator=g, device=device).to(BF16)
        self.attention = PagedAttention.initialize(q_heads, kv_heads, head_dim, lookahead)
        codes = E4M3 if eight_bits else None
        self.layers = [
            Layer(norm=norm(codes), qkv=Projection(matrix(hidden, (q_heads + 2 * kv_heads) * head_dim), eight_bits),
                  out=matrix(q_heads * head_dim, hidden), mlp_norm=norm(codes),
                  up=Projection(matrix(hidden, 4 * hidden), eight_bits), down=matrix(2 * hidden, hidden),
                  cache=PagedCache.allocate(pages, page_size, kv_heads, head_dim, dtype=cache, device=device))
            for _ in range(layers)
        ]
        self.norm = norm(None)
        self.head = matrix(hidden, vocab)

    def __call__(self, tokens: Tensor, table: Tensor, lengths: Tensor, cu_seqlens: Tensor | None = None,
                 last: Tensor | None = None) -> Tensor:
        """Logits after the new `tokens` `[n]`, which become the last ones of their requests'
        `lengths` cached tokens; of the rows `last` alone where that is given (a prompt's)."""
        hidden, residual = self.embedding[tokens], None
        for layer in self.layers:
            y, scales, total = layer.norm(hidden, residual)
            residual = hidden if total is None else total
            q, k, v = (layer.qkv(y, scales).view(-1, self.q_heads + 2 * self.kv_heads, self.head_dim)
                       .split([self.q_heads, self.kv_heads, self.kv_heads], dim=1))
            layer.cache.append(k, v, table, lengths, cu_seqlens)
            mixed = self.attention(q, layer.cache, table, lengths, cu_seqlens)
            y, scales, residual = layer.mlp_norm(mixed.flatten(1) @ layer.out, residual)
            gate, up = layer.up(y, scales).chunk(2, dim=-1)
            hidden = (F.silu(gate) * up) @ layer.down
        if last is not None:
            hidden, residual = hidden[last], residual[last]
        y, _, _ = self.norm(hidden, residual)
        return y @ self.head

    def swap_out(self, table: Tensor, lengths: Tensor) -> list[tuple[Tensor, Tensor]]:
        """The requests' cached keys and values of every layer, in host memory: their pages are free."""
        starts = F.pad(lengths.cumsum(0), (1, 0)).to(I32)
        total = int(starts[-1])
        return [tuple(x.cpu() for x in layer.cache.gather(table, starts, total)) for layer in self.layers]

    def swap_in(self, saved: list[tuple[Tensor, Tensor]], table: Tensor, lengths: Tensor) -> None:
        """Back into the pages of `table` (a bf16 cache then holds what it held)."""
        starts = F.pad(lengths.cumsum(0), (1, 0)).to(I32)
        for layer, (keys, values) in zip(self.layers, saved):
            layer.cache.append(keys.to(table.device), values.to(table.device), table, lengths, starts)

    def device_error(self) -> int:
        return self.attention.device_error() | max(layer.cache.device_error() for layer in self.layers)


def greedy_buffers(requests: int, timesteps: int, vocab: int, device) -> object:
    return workloads.sampling_buffers(requests, timesteps, vocab, device, 1,
                                      workloads.RequestParams([1.0], [1], [1.0], [0.0]), processors=False, greedy=True)


def drafts_from_history(history: list[list[int]], lookahead: int) -> list[list[int]]:
    """What followed the last earlier occurrence of each request's newest token, or that token again."""
    out = []
    for tokens in history:
        at = next((i for i in range(len(tokens) - 2, -1, -1) if tokens[i] == tokens[-1]), None)
        found = [] if at is None else tokens[at + 1 : at + 1 + lookahead]
        out.append((found + [tokens[-1]] * lookahead)[:lookahead])
    return out


def generate(model: Decoder, prompts: list[list[int]], table: Tensor, steps: int, lookahead: int = 0,
             draft=drafts_from_history) -> list[list[int]]:
    """`steps` calls after the prompts, with every request in each: greedy tokens, or with a
    `lookahead` that many drafted by `draft(history, lookahead)`, verified. Returns prompt and answer."""
    device, requests, vocab = table.device, len(prompts), model.head.size(1)
    buffers = greedy_buffers(requests, lookahead + 1, vocab, device)
    sampler = UnshardedFusedSingular.initialize(vocab, batch_size=requests)
    history = [list(p) for p in prompts]
    lengths = torch.tensor([len(p) for p in prompts], dtype=I32, device=device)
    starts = F.pad(lengths.cumsum(0), (1, 0)).to(I32)
    logits = model(torch.tensor(sum(history, []), device=device), table, lengths, starts, last=starts[1:].long() - 1)
    tokens = sampler.autoregressive(logits, buffers).tokens
    for tokens_of, new in zip(history, tokens.view(-1).tolist()):
        tokens_of.append(new)
    verifier = UnshardedFusedMultistep.initialize(vocab, lookahead, batch_size=requests) if lookahead else None
    for _ in range(steps):
        if verifier is None:
            lengths += 1
            tokens = sampler.autoregressive(model(tokens.view(-1).long(), table, lengths), buffers).tokens
            accepted = tokens.tolist()
        else:
            # the newest token and its drafts go in; lengths count all of them for this call, and
            # afterwards those whose tokens were kept: the newest and `offsets` drafts
            drafts = torch.tensor(draft(history, lookahead), dtype=I32, device=device)
            fed = torch.cat([tokens.view(-1, 1), drafts], dim=1)
            logits = model(fed.view(-1).long(), table, lengths + lookahead + 1)
            result = verifier(logits.view(requests, lookahead + 1, vocab), F.pad(drafts, (0, 1)).contiguous(), buffers)
            offsets = result.offsets.view(-1)
            lengths += offsets.to(I32) + 1
            tokens = result.tokens.view(requests, -1).gather(1, offsets.view(-1, 1).long())
            accepted = [row[: n + 1] for row, n in zip(result.tokens.view(requests, -1).tolist(), offsets.tolist())]
        for tokens_of, new in zip(history, accepted):
            tokens_of.extend(new)
    if error := model.device_error():
        raise RuntimeError(f"device error {error}: a page id or length outside the cache")
    return history


def page_table(requests: int, tokens: int, page_size: int, pages: int, device, seed: int = 0) -> Tensor:
    """Pages for `tokens` of every request, in no order, as a long-running pool would hand them out."""
    each = -(-tokens // page_size)
    if requests * each > pages:
        raise ValueError(f"{requests} requests of {tokens} tokens need {requests * each} pages, the cache has {pages}")
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: requests * each]
    return order.view(requests, each).to(I32).to(device)


def main(argv: list[str]) -> None:
    import argparse
    import time

    parser = argparse.ArgumentParser(prog="python -m sonic_sampler_b200.decode", description=__doc__.split("\n")[0])
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--prompt", type=int, default=200, help="longest prompt; the others are shorter")
    parser.add_argument("--steps", type=int, default=32)
    parser.add_argument("--lookahead", type=int, default=3)
    parser.add_argument("--cache", choices=("e4m3", "bf16"), default="e4m3")
    args = parser.parse_args(argv)
    if min(args.requests, args.prompt) < 1 or min(args.steps, args.lookahead) < 0:
        parser.error("--requests and --prompt must be positive, --steps and --lookahead not negative")
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 32000, (1 + (i + 1) * (args.prompt - 1) // args.requests,), generator=g).tolist()
               for i in range(args.requests)]
    room = args.prompt + (args.steps + 1) * (args.lookahead + 1)
    pages = args.requests * -(-room // 16)
    model = Decoder(pages=pages, lookahead=args.lookahead, cache=E4M3 if args.cache == "e4m3" else BF16,
                    eight_bits=args.cache == "e4m3")
    table = page_table(args.requests, room, 16, pages, "cuda")
    begin = time.perf_counter()
    history = generate(model, prompts, table, args.steps, args.lookahead)
    taken = time.perf_counter() - begin
    new = sum(len(h) - len(p) for h, p in zip(history, prompts))
    print(f"{args.requests} requests, {args.steps} steps: {new} tokens "
          f"({new / args.requests / (args.steps + 1):.2f} a call and request) in {taken:.2f} s, the first calls' set-up included")
    for p, h in list(zip(prompts, history))[:4]:
        print(f"  after {len(p)} tokens:", *h[len(p) : len(p) + 12])


if __name__ == "__main__":
    import sys

    main(sys.argv[1:])
