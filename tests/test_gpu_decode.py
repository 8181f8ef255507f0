"""The small decoder: norm, cache, attention and sampler composed as a served model composes them.

Its logits have a root mean square of about 1 (a normed row times columns of unit length). The same
tokens computed in calls of other shapes differ by roundings alone: some 20 a layer and pass to bf16
(2^-9 of a value in the root mean square, at most), so sqrt(2 * 40) * 2^-9 = 0.0175 for two layers and
two passes; the bound is twice that. In 8 bits such a difference also turns a few codes to their
neighbours: of relative differences of 0.01, a tenth cross a boundary, and a step is 0.06 to 0.12 of a
value, so up to sqrt(0.1) * 0.09 = 0.03 for each of 4 norms and 4 cached rows: 0.09 in all; the bound
is twice that."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from sonic_sampler_b200 import decode
from sonic_sampler_b200.decode import E4M3, I32, Decoder, generate, page_table

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
BOUND = {False: 0.035, True: 0.18}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    _abi.load_library()
    return torch.device("cuda", 0)


def _model(eight_bits, **kw):
    return Decoder(vocab=2048, hidden=256, layers=2, q_heads=4, kv_heads=2, head_dim=64, pages=64, page_size=16,
                   cache=E4M3 if eight_bits else BF16, eight_bits=eight_bits, **kw)


def _sequences(dev, lengths):
    g = torch.Generator().manual_seed(5)
    tokens = [torch.randint(0, 2048, (n,), generator=g) for n in lengths]
    return tokens, torch.tensor(lengths, dtype=I32, device=dev)


def _chunk(model, tokens, lengths, table):
    starts = F.pad(lengths.cumsum(0), (1, 0)).to(I32)
    return model(torch.cat(tokens).to(lengths.device), table, lengths, starts), starts


@pytest.mark.parametrize("eight_bits", [False, True])
@pytest.mark.parametrize("prompt", [1, 17])
def test_steps_agree_with_one_chunk(dev, eight_bits, prompt):
    model = _model(eight_bits)
    tokens, lengths = _sequences(dev, [prompt + 6] * 3)
    table = page_table(3, prompt + 6, 16, 64, dev)
    whole = _chunk(model, tokens, lengths, table)[0].view(3, prompt + 6, -1).float()
    fresh = _model(eight_bits)
    first, _ = _chunk(fresh, [t[:prompt] for t in tokens], torch.full_like(lengths, prompt), table)
    rows = [first.view(3, prompt, -1)]
    for i in range(prompt, prompt + 6):
        new = torch.stack([t[i] for t in tokens]).to(dev)
        rows.append(fresh(new, table, torch.full_like(lengths, i + 1)).unsqueeze(1))
    stepped = torch.cat(rows, dim=1).float()
    assert model.device_error() == fresh.device_error() == 0
    assert 0.5 < float(whole.square().mean().sqrt()) < 2.0
    assert float((whole - stepped).square().mean().sqrt()) < BOUND[eight_bits]


@pytest.mark.parametrize("lookahead,drafts", [(0, None), (3, "history"), (3, "right"), (3, "half")])
def test_generated_tokens_are_the_likeliest(dev, lookahead, drafts):
    """Every generated token is the likeliest of a pass over the whole answer, up to five times the
    difference of two logits' roundings, whatever is drafted; right drafts are kept."""
    model = _model(False, lookahead=lookahead)
    prompts = [t.tolist() for t in _sequences(dev, [1, 9, 40])[0]]
    table = page_table(3, 160, 16, 64, dev)
    kw = {}
    if drafts in ("right", "half"):
        answers = generate(_model(False), prompts, table, 110)

        def draft(history, n):
            # what the steps without drafts gave, every other call with a wrong second token
            out = [a[len(h) : len(h) + n] for h, a in zip(history, answers)]
            return [[t, t + 1 & 2047, u] if drafts == "half" and len(h) % 2 else [t, s, u] for (t, s, u), h in zip(out, history)]

        kw["draft"] = draft
    history = generate(model, prompts, table, 24, lookahead, **kw)
    new = sum(len(h) - len(p) for h, p in zip(history, prompts))
    assert all(len(h) >= len(p) + 25 for h, p in zip(history, prompts))
    if drafts in ("right", "half"):
        # a near tie may part the two ways, after which drafts are wrong
        assert new >= 3 * 25 + 24
    whole = _model(False)
    lengths = torch.tensor([len(h) - 1 for h in history], dtype=I32, device=dev)
    logits, starts = _chunk(whole, [torch.tensor(h[:-1]) for h in history], lengths, table)
    for b, (h, p) in enumerate(zip(history, prompts)):
        rows = logits[int(starts[b]) + len(p) - 1 : int(starts[b + 1])].float()
        chosen = torch.tensor(h[len(p) :], device=dev)
        assert (rows.amax(-1) - rows.gather(1, chosen[:, None])[:, 0] <= 5 * 2**0.5 * BOUND[False]).all()


def test_a_request_moved_to_the_host_and_to_other_pages_goes_on_unchanged(dev):
    model = _model(False)
    tokens, lengths = _sequences(dev, [33, 1, 16])
    table = page_table(3, 48, 16, 64, dev)
    _chunk(model, tokens, lengths, table)
    new = torch.tensor([3, 4, 5], device=dev)
    expect = model(new, table, lengths + 1)
    saved = model.swap_out(table, lengths)
    for layer in model.layers:
        layer.cache.keys.fill_(float("nan"))
        layer.cache.values.fill_(float("nan"))
    elsewhere = page_table(3, 48, 16, 64, dev, seed=9)
    assert not torch.equal(table, elsewhere)
    model.swap_in(saved, elsewhere, lengths)
    assert torch.equal(model(new, elsewhere, lengths + 1), expect)
    assert model.device_error() == 0


@pytest.mark.parametrize("cache", ["e4m3", "bf16"])
def test_the_command_runs(dev, capsys, cache):
    decode.main(["--requests", "3", "--prompt", "20", "--steps", "4", "--lookahead", "2", "--cache", cache])
    assert "3 requests, 4 steps" in capsys.readouterr().out
