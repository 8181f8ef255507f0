"""Cases of the decode-side operators: a paged key-value cache (quantised as it is written, read
back), the attention of new tokens over it, and the residual root-mean-square norm with an output
in 8 bits.

`run` computes a case either in plain torch operations (fp32 throughout, rounded once at the end)
or, with `own` set, through the public calls of `sonic_sampler_b200.interface`. `exact` restates
each operator in 64 bits.

Definitions. Request b has `lengths[b]` tokens in the cache, the last n_b of them new in this
call; its token at position p lies in page `page_table[b, p // page_size]`, slot `p % page_size`.
Query i of the request stands at position lengths[b] - n_b + i, sees the keys up to its own
position (at most `window` of them, where that is set), and is zero (log-sum-exp -inf) where it
sees none. A row quantised to e4m3 has the scale c / 448 with c = max(amax, 2^-60), and the codes
e4m3(x * (448 / c)). The norm takes r = x + residual in fp32 and gives r * rsqrt(mean(r^2) + eps)
* weight, and r rounded to the input type as the next residual.
"""

from __future__ import annotations

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
E4M3_MAX = 448.0
FLOOR = 2.0 ** -60
EPS = 1e-5


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------


def _attention(requests, tokens, shortest, longest, q_heads=32, kv_heads=8, head_dim=128, page_size=16, dtype="bf16",
               cache="bf16", window=0, ragged=False):
    return dict(op="attention", requests=requests, tokens=tokens, ragged=ragged, shortest=shortest, longest=longest,
                q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, cache=cache,
                window=window)


def _append(requests, tokens, shortest, longest, kv_heads=8, head_dim=128, page_size=16, dtype="bf16", cache="e4m3",
            ragged=False):
    return dict(op="append", requests=requests, tokens=tokens, ragged=ragged, shortest=shortest, longest=longest,
                kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, cache=cache)


def _gather(requests, shortest, longest, kv_heads=8, head_dim=128, page_size=16, dtype="bf16", cache="e4m3"):
    return dict(op="gather", requests=requests, tokens=1, ragged=False, shortest=shortest, longest=longest,
                kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, cache=cache)


def _norm(rows, hidden, dtype="bf16", out="e4m3", group=0, residual=True):
    return dict(op="norm", rows=rows, hidden=hidden, dtype=dtype, out=out, group=group, residual=residual)


def listed():
    return [
        # one request early in its answer: the call's latency
        {"name": "attention one short", **_attention(1, 1, 700, 700)},
        # a decode step of 64 requests of every length, a few just admitted
        {"name": "attention decode ragged", **_attention(64, 1, 1, 8192)},
        # a large batch over a quantised cache
        {"name": "attention decode e4m3", **_attention(128, 1, 2048, 16384, page_size=64, cache="e4m3")},
        # verification of up to 4 drafted tokens a request, 32 requests of other draft lengths;
        # the first requests have fewer tokens than queries
        {"name": "attention verify", **_attention(32, 5, 0, 4097, ragged=True)},
        # two long documents: few rows, so the work is split over the length
        {"name": "attention long e4m3", **_attention(2, 1, 100003, 131072, q_heads=64, cache="e4m3")},
        # a small model of another head layout: 7 query heads a key head, sliding window, odd page
        {"name": "attention window fp16", **_attention(128, 4, 5, 6001, q_heads=14, kv_heads=2, head_dim=64,
                                                       page_size=7, dtype="fp16", cache="fp16", window=1000)},
        # a decode step's 64 new tokens into a quantised cache
        {"name": "append decode e4m3", **_append(64, 1, 1, 1024)},
        # prompt chunks: 8 requests with 16000 new tokens in all
        {"name": "append prompt e4m3", **_append(8, 2000, 2000, 6000)},
        # reading back: a few requests on their way to the host, and whole contexts
        {"name": "gather few e4m3", **_gather(4, 10, 500)},
        {"name": "gather contexts e4m3", **_gather(16, 4000, 30001)},
        # the norm before a layer's projections: a decode step's rows, and a prompt chunk's
        {"name": "norm decode e4m3", **_norm(64, 4096)},
        {"name": "norm prompt e4m3", **_norm(16384, 8192, group=128)},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "append", "gather", "norm", "norm"))
    if op == "norm":
        hidden = _log_int(rng, 64, 16384)
        hidden = max(64, hidden if rng.random() < 0.3 else hidden // 64 * 64)
        dtype, out = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice(("e4m3", "e4m3", "same"))
        rows = _log_int(rng, 1, min(32768, (1 << 28) // (BYTES[dtype] * hidden)))
        return _norm(rows, hidden, dtype=dtype, out=out,
                     group=rng.choice((0, 128)) if out == "e4m3" else 0, residual=rng.random() < 0.8)
    kv_heads, head_dim = rng.choice((1, 2, 4, 8, 8)), rng.choice((64, 128, 128, 256))
    page_size = rng.choice((1, 7, 16, 16, 32, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    cache = rng.choice((dtype, "e4m3"))
    requests = _log_int(rng, 1, 256)
    # at most as many cached values as the largest listed case reads
    room = int((1 << 29) // (BYTES[cache] * kv_heads * head_dim * requests))
    if op == "attention":
        tokens, group = rng.choice((1, 1, 1, _log_int(rng, 2, 16))), rng.choice((1, 2, 3, 4, 7, 8, 16))
        # and at most 80 GFLOP, where many query rows share a key head
        room = min(room, 20 * 10 ** 9 // (tokens * group * kv_heads * head_dim * requests))
        longest = _log_int(rng, 1, max(2, min(131072, room)))
        return _attention(requests, tokens, rng.choice((0, 1, max(1, longest // 4), longest)), longest,
                          q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                          page_size=page_size, dtype=dtype, cache=cache, ragged=tokens > 1 and rng.random() < 0.5,
                          window=rng.choice((0, 0, _log_int(rng, 1, 4096))))
    if op == "append":
        tokens = rng.choice((1, _log_int(rng, 2, max(3, min(4096, 32768 // requests)))))
        return _append(requests, tokens, tokens, tokens + _log_int(rng, 1, max(2, min(2048, 65536 // requests))),
                       kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, cache=cache,
                       ragged=tokens > 1 and rng.random() < 0.5)
    longest = _log_int(rng, 1, max(2, min(32768, room // 2)))
    return _gather(requests, rng.choice((0, 1, max(1, longest // 4))), longest, kv_heads=kv_heads, head_dim=head_dim,
                   page_size=page_size, dtype=dtype, cache=cache)


def _sequences(case):
    """(length, new tokens) of each request: lengths spread over their range by their logarithm."""
    n, low, high = case["requests"], case["shortest"] + 1, case["longest"] + 1
    pairs = []
    for b in range(n):
        length = int(round(low * (high / low) ** ((b + 0.5) / n if n > 1 else 1.0))) - 1
        pairs.append((length, b % case["tokens"] + 1 if case["ragged"] else case["tokens"]))
    return pairs


def _visible(length, new, window):
    """First key that any of the request's queries sees."""
    return max(0, length - new - window + 1) if window else 0


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["hidden"], BYTES[case["dtype"]]
        moved = n * size * (3 if case["residual"] else 1) + case["hidden"] * size
        if case["out"] == "e4m3":
            groups = -(-case["hidden"] // case["group"]) if case["group"] else 1
            moved += n + 4 * case["rows"] * groups
        else:
            moved += n * size
        return {"bytes": moved, "flops": 6 * n}
    pairs = _sequences(case)
    row = case["kv_heads"] * case["head_dim"]
    scales = 8 * case["kv_heads"] if case["cache"] == "e4m3" else 0
    cached = 2 * row * BYTES[case["cache"]] + scales
    plain = 2 * row * BYTES[case["dtype"]]
    if case["op"] == "append":
        tokens = sum(new for _, new in pairs)
        return {"bytes": tokens * (cached + plain), "flops": 6 * tokens * row}
    if case["op"] == "gather":
        tokens = sum(length for length, _ in pairs)
        return {"bytes": tokens * (cached + plain), "flops": 2 * tokens * row}
    seen = sum(length - _visible(length, new, case["window"]) for length, new in pairs)
    queries = sum(new for _, new in pairs)
    scores = 0
    for length, new in pairs:
        for i in range(new):
            keys = max(0, length - new + i + 1)
            scores += min(keys, case["window"]) if case["window"] else keys
    out = queries * case["q_heads"] * (2 * case["head_dim"] * BYTES[case["dtype"]] + 4)
    return {"bytes": seen * cached + out, "flops": 4 * scores * case["q_heads"] * case["head_dim"]}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------


def _quantise(x):
    """e4m3 codes and scales of the rows of x (fp32)."""
    c = x.abs().amax(-1, keepdim=True).clamp(min=FLOOR)
    return (x * (E4M3_MAX / c)).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), (c / E4M3_MAX).squeeze(-1)


def _pages(case, pages, gen):
    """Pages of keys or values [pages, heads, slots, dim] with their scales (None in 16 bits).

    Channels differ in size, as the keys and values of a trained model do."""
    shape = (pages, case["kv_heads"], case["page_size"], case["head_dim"])
    spread = torch.empty(case["head_dim"], device="cuda").normal_(0.0, 0.7, generator=gen).exp_()
    data = torch.empty(shape, dtype=TYPES[case["cache"]], device="cuda")
    scales = torch.empty(shape[:3], device="cuda") if case["cache"] == "e4m3" else None
    step = max(1, (1 << 27) // (case["kv_heads"] * case["page_size"] * case["head_dim"]))
    for at in range(0, pages, step):
        x = torch.empty((min(step, pages - at), *shape[1:]), device="cuda").normal_(generator=gen) * spread
        if scales is None:
            data[at:at + step] = x.to(data.dtype)
        else:
            data[at:at + step], scales[at:at + step] = _quantise(x)
    return data, scales


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.empty(shape, device="cuda").normal_(generator=gen)

    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        # a residual stream has a few channels far larger than the others
        spread = torch.where(torch.rand(hidden, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
        state = {"case": case, "x": normal(rows, hidden).to(dtype),
                 "residual": (normal(rows, hidden) * spread).to(dtype) if case["residual"] else None,
                 "weight": (1.0 + 0.2 * normal(hidden)).to(dtype)}
        if own:
            from sonic_sampler_b200.interface import ResidualNorm

            state["norm"] = ResidualNorm(state["weight"], eps=EPS, dtype=E4M3 if case["out"] == "e4m3" else None,
                                         group=case["group"] or None)
        return state

    order = random.Random(seed)
    pairs = _sequences(case)
    order.shuffle(pairs)
    counts = [-(-length // case["page_size"]) for length, _ in pairs]
    spare = sum(counts) // 16 + 1
    pages = sum(counts) + spare
    free = torch.randperm(pages, device="cuda", generator=gen, dtype=torch.int32)
    # row b holds its own pages, then page 0 (never read)
    width = max(1, max(counts))
    table = torch.zeros(len(pairs), width, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table[held] = free[:sum(counts)]
    offsets = [0]
    for _, new in pairs:
        offsets.append(offsets[-1] + new)
    state = {"case": case, "table": table,
             "lengths": torch.tensor([length for length, _ in pairs], dtype=torch.int32, device="cuda"),
             "cu": torch.tensor(offsets, dtype=torch.int32, device="cuda") if case["ragged"] else None,
             "tokens": case["tokens"]}
    state["keys"], state["key_scales"] = _pages(case, pages, gen)
    state["values"], state["value_scales"] = _pages(case, pages, gen)
    if case["op"] == "attention":
        # a few heads attend sharply, the others broadly
        sharp = torch.where(torch.rand(case["q_heads"], 1, device="cuda", generator=gen) < 0.25, 3.0, 0.7)
        state["q"] = (normal(offsets[-1], case["q_heads"], case["head_dim"]) * sharp).to(dtype)
    elif case["op"] == "append":
        # keys and values as they come out of one projection: [tokens, keys | values]
        fused = normal(offsets[-1], 2, case["kv_heads"], case["head_dim"]) * (0.5 + normal(offsets[-1], 2, case["kv_heads"], 1).exp())
        state["new"] = fused.to(dtype)
    else:
        starts = [0]
        for length, _ in pairs:
            starts.append(starts[-1] + length)
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        state["total"] = starts[-1]
    if own:
        from sonic_sampler_b200.interface import PagedAttention, PagedCache

        state["cache"] = PagedCache(keys=state["keys"], values=state["values"], key_scales=state["key_scales"],
                                    value_scales=state["value_scales"])
        if case["op"] == "attention":
            state["attention"] = PagedAttention.initialize(
                q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"], lookahead=case["tokens"] - 1)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "gather": _plain_gather,
                "norm": _plain_norm}[case["op"]](state)
    if case["op"] == "attention":
        out, lse = state["attention"](state["q"], state["cache"], state["table"], state["lengths"], cu_seqlens=state["cu"],
                                      window=case["window"] or None, logsumexp=True)
        return {"out": out, "lse": lse}
    if case["op"] == "append":
        state["cache"].append(state["new"][:, 0], state["new"][:, 1], state["table"], state["lengths"], cu_seqlens=state["cu"])
        return _cache_state(state)
    if case["op"] == "gather":
        keys, values = state["cache"].gather(state["table"], state["starts"], state["total"], dtype=TYPES[case["dtype"]])
        return {"keys": keys, "values": values}
    out, scales, residual = state["norm"](state["x"], state["residual"])
    return _present({"out": out, "scales": scales, "residual": residual})


def _present(outputs):
    return {k: v for k, v in outputs.items() if v is not None}


def _cache_state(state):
    return _present({k: state[k] for k in ("keys", "values", "key_scales", "value_scales")})


def _pages_of(data, scales, table):
    """The pages of every request, in fp32, as [requests, heads, positions, dim]."""
    if scales is None:
        x = data[table].float()
    else:
        x = data.view(torch.uint8)[table].view(E4M3).float() * scales[table].unsqueeze(-1)
    b, p, h, s, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * s, d)


def _plain_attention(state):
    case, q, lengths = state["case"], state["q"], state["lengths"].long()
    b, (n, hq, d), h, most = lengths.numel(), q.shape, case["kv_heads"], case["tokens"]
    group = hq // h
    steps = torch.arange(most, device=q.device)
    if state["cu"] is None:
        new = torch.full_like(lengths, most)
        first = torch.arange(b, device=q.device) * most
    else:
        cu = state["cu"].long()
        new, first = cu[1:] - cu[:-1], cu[:-1]
    live = steps < new[:, None]                                            # [b, most]
    rows = (first[:, None] + steps).clamp(max=n - 1)
    x = q[rows].float().view(b, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * group, d)
    keys = _pages_of(state["keys"], state["key_scales"], state["table"])
    scores = torch.matmul(x, keys.transpose(-1, -2)) * (1.0 / math.sqrt(d))  # [b, h, most * group, positions]
    del keys
    at = torch.arange(scores.size(-1), device=q.device)
    position = (lengths - new)[:, None] + steps                            # [b, most]
    sees = at <= position[..., None]
    if case["window"]:
        sees &= at > position[..., None] - case["window"]
    scores = scores.view(b, h, most, group, -1).masked_fill(~sees[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    values = _pages_of(state["values"], state["value_scales"], state["table"])
    out = torch.matmul(weights.view(b, h, most * group, -1), values).view(b, h, most, group, d)
    out = out / torch.where(total == 0.0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(-1)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, most, hq, d)[live]
    return {"out": out.to(q.dtype), "lse": lse.permute(0, 2, 1, 3).reshape(b, most, hq)[live]}


def _new_positions(state):
    """(page, slot) of every new token of the call."""
    lengths, n, size = state["lengths"].long(), state["new"].size(0), state["keys"].size(2)
    rows = torch.arange(n, device=lengths.device)
    if state["cu"] is None:
        request, step, new = rows // state["tokens"], rows % state["tokens"], state["tokens"]
        position = lengths[request] - new + step
    else:
        cu = state["cu"].long()
        request = torch.searchsorted(cu, rows, right=True) - 1
        position = lengths[request] - cu[request + 1] + rows
    return state["table"][request, position // size].long(), position % size


def _plain_append(state):
    page, slot = _new_positions(state)
    for j, name in enumerate(("keys", "values")):
        x, scales = state["new"][:, j], state[name[:-1] + "_scales"]
        if scales is None:
            state[name][page, :, slot] = x
        else:
            codes, scale = _quantise(x.float())
            state[name].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            scales[page, :, slot] = scale
    return _cache_state(state)


def _plain_gather(state):
    case, starts, size = state["case"], state["starts"].long(), state["keys"].size(2)
    rows = torch.arange(state["total"], device=starts.device)
    request = torch.searchsorted(starts, rows, right=True) - 1
    position = rows - starts[request]
    page, slot = state["table"][request, position // size].long(), position % size
    found = {}
    for name in ("keys", "values"):
        scales = state[name[:-1] + "_scales"]
        if scales is None:
            found[name] = state[name][page, :, slot].to(TYPES[case["dtype"]])
        else:
            x = state[name].view(torch.uint8)[page, :, slot].view(E4M3).float()
            found[name] = (x * scales[page, :, slot].unsqueeze(-1)).to(TYPES[case["dtype"]])
    return found


def _plain_norm(state):
    case, x = state["case"], state["x"]
    r = x.float() if state["residual"] is None else x.float() + state["residual"].float()
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * state["weight"].float()
    residual = None if state["residual"] is None else r.to(x.dtype)
    if case["out"] != "e4m3":
        return _present({"out": y.to(x.dtype), "residual": residual})
    rows, hidden = y.shape
    group = case["group"] or hidden
    groups = -(-hidden // group)
    padded = torch.nn.functional.pad(y, (0, groups * group - hidden)).view(rows, groups, group)
    codes, scales = _quantise(padded)
    return _present({"out": codes.view(rows, groups * group)[:, :hidden].contiguous(), "scales": scales, "residual": residual})


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------


def _e4m3_64(v):
    """Values of e4m3 nearest to v (fp64), ties to even."""
    e = torch.frexp(v).exponent.to(torch.float64) - 1.0
    quantum = torch.exp2(torch.clamp(e, min=-6.0) - 3.0)
    return torch.clamp(torch.round(v / quantum) * quantum, -E4M3_MAX, E4M3_MAX)


def _quantise_64(x):
    top = torch.clamp(x.abs().max(-1, keepdim=True).values, min=FLOOR)
    return _e4m3_64(x * E4M3_MAX / top), top.squeeze(-1) / E4M3_MAX


def _cached_64(state, name, request, length):
    """Rows [0, length) of a request, [heads, length, dim] in fp64."""
    size, data, scales = state[name].size(2), state[name], state[name[:-1] + "_scales"]
    position = torch.arange(length, device=data.device)
    page, slot = state["table"][request].long()[position // size], position % size
    if scales is None:
        x = data[page, :, slot].double()
    else:
        x = data.view(torch.uint8)[page, :, slot].view(E4M3).double() * scales[page, :, slot].double()[..., None]
    return x.transpose(0, 1)


def _exact_attention(case, state):
    q, h, d = state["q"], case["kv_heads"], case["head_dim"]
    group = case["q_heads"] // h
    lengths = state["lengths"].tolist()
    cu = [i * case["tokens"] for i in range(len(lengths) + 1)] if state["cu"] is None else state["cu"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths):
        new = cu[b + 1] - cu[b]
        if not length:
            continue
        keys, values = _cached_64(state, "keys", b, length), _cached_64(state, "values", b, length)
        for i in range(new):
            last = length - new + i
            first = max(0, last - case["window"] + 1) if case["window"] else 0
            if last < 0:
                continue
            k, v = keys[:, first:last + 1], values[:, first:last + 1]
            row = q[cu[b] + i].double().view(h, group, d)
            s = torch.einsum("hgd,hkd->hgk", row, k) / math.sqrt(d)
            total = torch.logsumexp(s, -1)
            out[cu[b] + i] = torch.einsum("hgk,hkd->hgd", torch.exp(s - total[..., None]), v).reshape(-1, d)
            lse[cu[b] + i] = total.reshape(-1)
    return {"out": out, "lse": lse}


def _exact_append(case, state):
    found = {k: v.double() for k, v in _cache_state(state).items()}
    lengths = state["lengths"].tolist()
    cu = [i * case["tokens"] for i in range(len(lengths) + 1)] if state["cu"] is None else state["cu"].tolist()
    table = state["table"].long()
    for b, length in enumerate(lengths):
        new = cu[b + 1] - cu[b]
        position = torch.arange(length - new, length, device=table.device)
        page, slot = table[b][position // case["page_size"]], position % case["page_size"]
        rows = state["new"][cu[b]:cu[b + 1]].double()
        for j, name in enumerate(("key", "value")):
            if case["cache"] == "e4m3":
                codes, scale = _quantise_64(rows[:, j])
                found[name + "s"][page, :, slot] = codes
                found[name + "_scales"][page, :, slot] = scale
            else:
                found[name + "s"][page, :, slot] = rows[:, j]
    return found


def _exact_gather(case, state):
    lengths = state["lengths"].tolist()
    return {name: torch.cat([_cached_64(state, name, b, n).transpose(0, 1) for b, n in enumerate(lengths)])
            for name in ("keys", "values")}


def _exact_norm(case, state):
    r = state["x"].double()
    if state["residual"] is not None:
        r = r + state["residual"].double()
    y = r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS) * state["weight"].double()
    found = {"out": y, "residual": r if state["residual"] is not None else None}
    if case["out"] == "e4m3":
        step = case["group"] or case["hidden"]
        parts = [_quantise_64(y[:, at:at + step]) for at in range(0, case["hidden"], step)]
        found["out"] = torch.cat([codes for codes, _ in parts], -1)
        found["scales"] = torch.stack([scale for _, scale in parts], -1)
    return _present(found)


def exact(case, seed):
    if case["op"] == "attention" and sum(new for _, new in _sequences(case)) > 4096:
        return None  # over 20 seconds
    state = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "gather": _exact_gather,
            "norm": _exact_norm}[case["op"]](case, state)
