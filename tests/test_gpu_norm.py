"""The residual norm against its 64-bit restatement: every type, aligned and odd row lengths, rows
in one warp and in many, outputs in 16, 32 and 8 bits."""

from __future__ import annotations

import math

import pytest
import torch

import decode_reference as ref
from decode_reference import E4M3

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from sonic_sampler_b200 import _abi

    _abi.load_library()
    return torch.device("cuda", 0)


def _inputs(dev, rows, hidden, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=gen).to(dtype).to(dev)
    residual = (torch.randn(rows, hidden, generator=gen) * 10 ** (torch.rand(hidden, generator=gen) * 2 - 1)).to(dtype).to(dev)
    weight = (1 + 0.3 * torch.randn(hidden, generator=gen)).to(dtype).to(dev)
    return x, residual, weight


def _check(out, scales, r_out, x, residual, weight, eps, group):
    hidden = x.size(-1)
    r, y = ref.norm(x, residual, weight, eps)
    # fp32: one rounding of the sum, hidden / 2 roundings of the squares' sum at most (halved under
    # the root), a handful of the factors
    relative = 2.0 ** -24 * (hidden / 2 + 16)
    slack = relative * y.abs() + 2.0 ** -24 * (r.abs() + x.double().abs()) * (y.abs() / r.abs().clamp(min=1e-300))
    if residual is not None:
        assert ((r_out.double() - r).abs() <= r.abs() * ref.EPS[x.dtype] * 1.01 + ref.TINY[x.dtype] + 2.0 ** -24 * r.abs()).all()
    else:
        assert r_out is None
    if out.dtype != E4M3:
        assert out.dtype == x.dtype and scales is None
        assert ((out.double() - y).abs() <= slack + y.abs() * ref.EPS[x.dtype] * 1.01 + ref.TINY[x.dtype]).all()
        return
    step = group or hidden
    groups = -(-hidden // step)
    assert scales.shape == (*x.shape[:-1], groups) and scales.dtype == F32
    for i in range(groups):
        part, err = y[:, i * step:(i + 1) * step], slack[:, i * step:(i + 1) * step]
        top = part.abs().amax(-1).clamp(min=ref.FLOOR)
        worst = err.amax(-1) + 2.0 ** -23 * top
        assert ((scales[:, i].double() * 448.0 - top).abs() <= worst).all()
        # the code is the nearest to y / scale, up to the errors of both
        quotient = part / (top[:, None] / 448.0)
        off = (out[:, i * step:(i + 1) * step].float().double() - quotient).abs()
        doubt = (err + part.abs() * (worst / top)[:, None]) * 448.0 / top[:, None] + 2.0 ** -22 * quotient.abs()
        assert (off <= ref.e4m3_step(quotient.abs() + doubt) * 0.5 + doubt).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out,group", [(None, None), (E4M3, None), (E4M3, 128)])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (5, 64), (2, 127), (9, 128), (4, 136), (3, 1000), (7, 1024), (300, 1023),
                                         (2, 4096), (400, 4096), (3, 5001), (350, 5120), (2, 16384), (300, 8192), (2, 32768),
                                         (2, 32767)])
def test_norm(dev, dtype, out, group, rows, hidden):
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, rows, hidden, dtype, rows + hidden)
    norm = ResidualNorm(weight, eps=1e-5, dtype=out, group=group)
    y, scales, r = norm(x, residual)
    _check(y, scales, r, x, residual, weight, 1e-5, group)
    y, scales, r = norm(x)
    _check(y, scales, r, x, None, weight, 1e-5, group)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("out,group", [(None, None), (E4M3, 128)])
def test_strides_alignment_and_shapes(dev, dtype, out, group):
    """Rows of a wider tensor, rows that start off 16-byte boundaries, leading dimensions."""
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, 6, 512, dtype, 1)
    norm = ResidualNorm(weight, eps=1e-6, dtype=out, group=group)
    want = norm(x, residual)
    for shift, width in ((0, 520), (8, 520), (3, 517), (1, 513)):
        wx, wr = (torch.full((6, width), math.nan, dtype=dtype, device=dev) for _ in range(2))
        wx[:, shift:shift + 512], wr[:, shift:shift + 512] = x, residual
        got = norm(wx[:, shift:shift + 512], wr[:, shift:shift + 512])
        _check(*got, x, residual, weight, 1e-6, group)
        # the residual in place, outputs inside wider tensors
        into = torch.zeros(6, width, dtype=out or dtype, device=dev)
        norm(x, wr[:, shift:shift + 512], residual_out=wr[:, shift:shift + 512], out=into[:, shift:shift + 512])
        assert torch.equal(wr[:, shift:shift + 512], want[2])
        keep = torch.ones(width, dtype=torch.bool, device=dev)
        keep[shift:shift + 512] = False
        assert torch.isnan(wr[:, keep]).all() and not into.float()[:, keep].any()
    shaped = norm(x.view(2, 3, 512), residual.view(2, 3, 512))
    assert shaped[0].shape == (2, 3, 512) and torch.equal(shaped[2].view(6, 512), want[2])


@pytest.mark.parametrize("group", [None, 128])
def test_edges(dev, group):
    """All-zero rows, rows with an infinity or a NaN, and their neighbours."""
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, 5, 512, BF16, 2)
    x[1], residual[1] = 0.0, 0.0
    x[2, 200] = math.nan
    x[3, 10] = math.inf
    norm = ResidualNorm(weight, eps=0.0, dtype=E4M3, group=group)
    y, scales, r = norm(x, residual)
    assert torch.isfinite(y[[0, 4]].float()).all() and torch.isfinite(scales[[0, 4]]).all()
    # 0 / sqrt(0): NaN by the formula with eps = 0; zeros with any other
    assert torch.isnan(y[1].float()).all()
    assert torch.isnan(y[2].float() * scales[2].repeat_interleave(512 // scales.size(1))).all()
    assert torch.isnan(y[3, 10].float() * scales[3, 0])
    y, scales, _ = ResidualNorm(weight, eps=1e-6, dtype=E4M3, group=group)(x, residual)
    assert not y[1].float().any() and torch.isfinite(scales[1]).all() and (scales[1] > 0).all()


def test_no_rows_streams_and_graphs(dev):
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, 40, 768, BF16, 3)
    norm = ResidualNorm(weight, dtype=E4M3, group=128)
    y, scales, r = norm(x[:0], residual[:0])
    assert y.shape == (0, 768) and scales.shape == (0, 6)
    want = norm(x, residual)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = norm(x, residual)
    stream.synchronize()
    static = [t.clone() for t in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm(x, residual, out=static[0], scales=static[1], residual_out=static[2])
    for t in static:
        t.view(torch.uint8).zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, static):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8))


def test_refusals(dev):
    from sonic_sampler_b200 import _abi
    from sonic_sampler_b200.interface import ResidualNorm

    x, residual, weight = _inputs(dev, 4, 256, BF16, 4)
    norm = ResidualNorm(weight)
    for message, args in (("columns", (x[:, :128],)), ("bfloat16", (x, residual.half())), ("CUDA tensors only", (x.cpu(),)),
                          ("residual", (x, residual[:2])), ("weight", (x.half(),)), ("unit inner stride", (x.T.contiguous().T,))):
        with pytest.raises(ValueError, match=message):
            norm(*args)
    with pytest.raises(ValueError, match="out"):
        norm(x, out=torch.empty(4, 256, dtype=F16, device=dev))
    with pytest.raises(ValueError, match="scales"):
        norm(x, out=torch.empty(4, 256, dtype=E4M3, device=dev), scales=torch.empty(4, 2, device=dev))
    with pytest.raises(ValueError, match="group"):
        ResidualNorm(weight, dtype=E4M3, group=64)
    with pytest.raises(ValueError, match="group"):
        ResidualNorm(weight, group=128)
    with pytest.raises(ValueError, match="dtype"):
        ResidualNorm(weight, dtype=F32)
    with pytest.raises(ValueError, match="eps"):
        ResidualNorm(weight, eps=-1.0)
    wide = torch.ones(40000, dtype=BF16, device=dev)
    with pytest.raises(_abi.SonicError, match="32768"):
        ResidualNorm(wide)(wide[None])
