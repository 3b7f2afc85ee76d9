"""4-bit weights on the GPU: the quantizer, packing and dense weight bit for bit
against the oracle, ``linear4`` against 64-bit sums.

Tolerance of a sum: the products value * x are exact in fp32 (2 + 8 significant
bits) and so is a weight's scale; a group's sum has at most ``group`` additions,
the scaled sums, the waves' parts and the splits of K together K / 32 + 32 more, each off by at most 2^-23
of the magnitudes added so far (twice a rounding's half step, for adders that cut
instead of rounding): (group + K / 32 + 32) 2^-23 sum |x| |w|.  The output adds half
a step of its type, and with a residual the linear's own rounding to that type
comes before."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import activations, bf16_gpu, to_np
from oracle import drafting_oracle as D
from oracle import quantization_oracle as O
from pageserve_amd import QuantizedWeight4, linear4

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _weights(seed, n, k):
    return (np.random.default_rng(seed).standard_normal((n, k)) * 0.02).astype(np.float32)


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32).cpu()


@pytest.mark.parametrize("n,k,group", [(1, 16, 32), (16, 128, 128), (17, 144, 64), (33, 896, 32), (130, 272, 128),
                                       (5, 2048, 64), (300, 48, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantizer_and_dense_match_the_oracle(gpu, n, k, group, dtype):
    w = torch.from_numpy(_weights(n + k + group, n, k)).to(dtype)
    w[0] = 0
    w[-1, :8] = torch.tensor([0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0, 6.0]).to(dtype)  # ties
    codes, scale = D.quantize4(w.float().numpy(), group)
    qw = QuantizedWeight4(w.to(gpu), group)
    assert np.array_equal(qw.codes.cpu().numpy(), codes)
    assert np.array_equal(qw.scale.float().cpu().numpy(), scale)
    cpu = QuantizedWeight4(w, group)
    assert torch.equal(qw.qp.cpu(), cpu.qp) and torch.equal(_bits(qw.sp), _bits(cpu.sp))  # padding too
    want = torch.from_numpy(D.dense4(codes, scale, group)).to(dtype)
    assert qw.dense().dtype == dtype and torch.equal(qw.dense().cpu(), want)


def test_quantizer_on_views_and_not_finite_weights(gpu):
    w = torch.from_numpy(_weights(8, 40, 320))
    w[3, 5], w[7, 70], w[9, 130] = float("nan"), float("inf"), -float("inf")
    full = torch.empty(40 * 320 + 1, device=gpu)
    shifted = full[1:].view(40, 320).copy_(w)       # 4-byte aligned
    strided = torch.empty(320, 40, device=gpu).t().copy_(w)
    codes, scale = D.quantize4(w.numpy(), 64)
    for src in (w.to(gpu), shifted, strided):
        qw = QuantizedWeight4(src, 64)
        assert np.array_equal(qw.codes.cpu().numpy(), codes)
        assert np.array_equal(qw.scale.float().cpu().numpy(), scale, equal_nan=True)
    assert torch.isnan(qw.dense()[3, :64]).all() and torch.isfinite(qw.dense()[3, 64:]).all()


def _case(gpu, m, n, k, group, seed=0):
    codes, scale = D.quantize4(_weights(seed + n, n, k), group)
    qw = QuantizedWeight4.from_codes(torch.from_numpy(codes).to(gpu), torch.from_numpy(scale).to(gpu).bfloat16(), group)
    return qw, D.dense4(codes, scale, group), activations(seed + m, m, k)


def _check(y, w, x, group, dtype, bias=None, residual=None, what=""):
    lin = x.astype(np.float64) @ w.T + (0 if bias is None else bias)
    size = np.abs(x).astype(np.float64) @ np.abs(w).T + (0 if bias is None else np.abs(bias))
    tol = (group + w.shape[1] / 32 + 32) * 2.0 ** -23 * size
    want = lin
    if residual is not None:
        tol = tol + U[dtype] * (np.abs(lin) + tol)
        want = lin + residual
    tol = tol + U[dtype] * (np.abs(want) + tol)
    got = to_np(y).astype(np.float64)
    assert got.shape == want.shape
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), f"{what}: {off.max():.3g} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 16, 32), (1, 16, 128, 128), (3, 17, 144, 64), (1, 2048, 2048, 128), (5, 1000, 896, 32), (16, 100, 4864, 64),
    (8, 896, 896, 128), (9, 896, 896, 128), (2, 2048, 11008, 32), (17, 48, 272, 32), (32, 896, 4864, 128), (30, 33, 1040, 64),
    (33, 250, 2048, 64), (64, 128, 528, 128), (65, 40, 160, 32), (130, 513, 640, 64), (1, 9000, 256, 64),
    (24, 40000, 256, 32), (4, 8, 32768, 32),
    # whole tiles for few tokens, four tiles a workgroup, K split over workgroups
    (8, 8191, 144, 128), (16, 8209, 272, 32), (31, 8300, 528, 128), (61, 8190, 400, 64),
    (9, 100, 11008, 64), (16, 2048, 11008, 128), (30, 50, 8208, 32), (60, 896, 4864, 64), (200, 70, 11024, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(gpu, m, n, k, group, dtype):
    qw, w, x = _case(gpu, m, n, k, group)
    _check(linear4(bf16_gpu(x, gpu), qw, out_dtype=dtype), w, x, group, dtype, what="plain")
    rng = np.random.default_rng(m + n)
    bias = O.round_to_bf16(rng.standard_normal(n).astype(np.float32))
    res = O.round_to_bf16(rng.standard_normal((m, n)).astype(np.float32))
    y = linear4(bf16_gpu(x, gpu), qw, bf16_gpu(bias, gpu), out_dtype=dtype, residual=bf16_gpu(res, gpu))
    _check(y, w, x, group, dtype, bias, res, "bias and residual")


def test_out_in_place_shapes_and_views(gpu):
    qw, w, x = _case(gpu, 6, 144, 208, 64)
    xt = bf16_gpu(x, gpu)
    y = linear4(xt, qw)
    assert torch.equal(linear4(xt.view(2, 3, 208), qw), y.view(2, 3, 144))
    wide = torch.zeros(6, 211, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:] = xt
    assert torch.equal(linear4(wide[:, 3:], qw), y)
    res = bf16_gpu(activations(2, 6, 144), gpu)
    want = linear4(xt, qw, residual=res)
    assert linear4(xt, qw, residual=res, out=res) is not None and torch.equal(res, want)
    assert torch.equal(qw.linear(xt), y)
    assert linear4(xt[:0], qw).shape == (0, 144)
    assert linear4(xt.view(6, 1, 208)[:, :0], qw).shape == (6, 0, 144)
    empty = QuantizedWeight4(torch.zeros(0, 64, device=gpu), 32)
    assert linear4(xt[:, :64], empty).shape == (6, 0) and empty.dense().shape == (0, 64)


def test_no_columns(gpu):
    qw = QuantizedWeight4(torch.zeros(20, 0, device=gpu), 64)
    x, bias = torch.zeros(3, 0, dtype=torch.bfloat16, device=gpu), torch.arange(20, device=gpu).bfloat16()
    assert qw.dense().shape == (20, 0) and qw.scale.shape == (20, 0) and qw.codes.shape == (20, 0)
    assert not linear4(x, qw).any()
    res = torch.ones(3, 20, dtype=torch.bfloat16, device=gpu)
    assert torch.equal(linear4(x, qw, bias, residual=res), (bias + 1).expand(3, 20))
    assert linear4(x[0], qw).shape == (20,)


def test_two_streams_at_once(gpu):
    """Calls that need a workspace, on two streams with nothing between them: each its own."""
    qw, _, x = _case(gpu, 20, 512, 11008, 64)
    xs = [bf16_gpu(activations(s, 20, 11008), gpu) for s in range(2)]
    want = [linear4(t, qw) for t in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(linear4(xs[i], qw))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_tokens_do_not_touch_each_other(gpu):
    """K ends inside a block: the next row's first values (not finite here) are not read as
    this row's, and a token's infinity stays its own."""
    for m, k in [(3, 144), (20, 144), (40, 16)]:
        qw, w, x = _case(gpu, m, 40, k, 32)
        xt = bf16_gpu(x, gpu)
        want = linear4(xt, qw)
        xt[1] = float("nan")
        xt[2, 0] = float("inf")
        y = linear4(xt, qw)
        rows = [0] + list(range(3, m))
        assert torch.equal(y[rows], want[rows]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()


def test_in_place_residual_of_a_split_sum(gpu):
    qw, w, x = _case(gpu, 20, 80, 11008, 64)
    xt, res = bf16_gpu(x, gpu), bf16_gpu(activations(2, 20, 80), gpu)
    want = linear4(xt, qw, residual=res)
    linear4(xt, qw, residual=res, out=res)
    assert torch.equal(res, want)


@pytest.mark.parametrize("m,n,k", [(5, 512, 2048), (20, 256, 11008)])
def test_streams_and_graph_replays(gpu, m, n, k):
    qw, w, x = _case(gpu, m, n, k, 128)
    xt = bf16_gpu(x, gpu)
    want = linear4(xt, qw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = linear4(xt, qw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = linear4(xt, qw)
        z = QuantizedWeight4(y.float(), 32).dense()
    for seed in range(3):
        xt.copy_(bf16_gpu(activations(seed, m, k), gpu))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, linear4(xt, qw)) and torch.equal(z, QuantizedWeight4(y.float(), 32).dense())


def test_refusals(gpu):
    qw, _, x = _case(gpu, 2, 32, 64, 32)
    xt = bf16_gpu(x, gpu)
    with pytest.raises(TypeError, match="bf16 activations"):
        linear4(xt.float(), qw)
    with pytest.raises(ValueError, match="features"):
        linear4(xt[:, :48], qw)
    with pytest.raises(ValueError, match="weight on"):
        linear4(xt.cpu(), qw)
    with pytest.raises(TypeError, match="out_dtype"):
        linear4(xt, qw, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bias"):
        linear4(xt, qw, torch.zeros(31, dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError, match="residual"):
        linear4(xt, qw, residual=torch.zeros(3, 32, dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError, match="out must"):
        linear4(xt, qw, out=torch.zeros(2, 32, device=gpu))
    room = torch.zeros(5 * 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError, match="share memory with the input"):
        linear4(room[:128].view(2, 64), qw, out=room[120:184].view(2, 32))
    with pytest.raises(ValueError, match="residual itself"):
        linear4(xt, qw, residual=room[:64].view(2, 32), out=room[8:72].view(2, 32))
    with pytest.raises(ValueError, match="residual itself"):
        linear4(xt, qw, residual=room[:64].view(2, 32), out=room[:128].view(torch.float32).view(2, 32),
                out_dtype=torch.float32)


def test_out_in_the_weight_or_the_bias_is_refused(gpu):
    qw, _, x = _case(gpu, 1, 64, 64, 32)
    xt = bf16_gpu(x, gpu)
    room = torch.zeros(200, dtype=torch.bfloat16, device=gpu)
    codes = qw.qp.clone()
    for kw in (dict(bias=room[:64], out=room[32:96].view(1, 64)), dict(out=qw.qp.view(torch.bfloat16)[64:128].view(1, 64)),
               dict(out=qw.sp[8:72].view(1, 64)), dict(out=qw.sp[:128].view(torch.float32).view(1, 64), out_dtype=torch.float32)):
        with pytest.raises(ValueError, match="weight or the bias"):
            linear4(xt, qw, **kw)
    assert torch.equal(qw.qp, codes)
    y = linear4(xt, qw, bias=room[:64], out=room[64:128].view(1, 64))
    assert torch.equal(y, linear4(xt, qw))
