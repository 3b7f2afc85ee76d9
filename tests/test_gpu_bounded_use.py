"""Sums of weights on other streams, and eviction of rows far into a large cache: what is written,
number by number (tests/test_gpu_evict.py: the bound of sums)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bounded import Batch
from oracle import window_oracle as W
from pageserve_amd import KVCache4, accumulate_weights, evict_tokens, read_kv4, window_attention, window_attention4
from test_gpu_evict import check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [2, 70, 600])
def test_sums_on_other_streams(gpu, tokens, bits):
    """Two streams at once, each step's attention and sums behind the other: every step's sums"""
    b = Batch(tokens, [tokens + 100, 200, 40, tokens], [tokens, 1, 0, tokens], 16, 2, 128, 16, torch.bfloat16, bits)
    args, seen = b.args(gpu), {"window": 90, "sinks": 4}
    start = torch.rand(b.blocks, b.bs, device=gpu)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams * 3:
        with torch.cuda.stream(s):
            _, lse = (window_attention4 if bits == 4 else window_attention)(*args, return_lse=True, **seen)
            sums = start.clone()
            accumulate_weights(args[0], args[1], *args[-3:], lse, sums, **seen)
            got.append((lse, sums))
    for s in streams:
        s.synchronize()
    for lse, sums in got:
        want, far = W.accumulate(start.cpu().numpy(), b.q.double().numpy(), b.dense()[0], b.tables, b.lens, b.offsets,
                                 lse.double().cpu().numpy(), b.dim ** -0.5, None, **seen)
        check_weights(b, sums, want, far)
        assert torch.equal(sums, got[0][1])


@pytest.mark.parametrize("bits,dim", [(16, 128), (16, 64), (4, 128), (4, 64)])
def test_eviction_moves_rows_beyond_32_bits(gpu, bits, dim):
    """Blocks whose bytes and elements lie beyond 2^32 and 2^31, and others at the front"""
    bs, kv, lens, budget = 64, 2, [300, 77], [60, 70]
    high = (1 << 32) // (bs * kv * (2 * dim if bits == 16 else dim // 2)) + 100
    blocks = high + 9
    tables = torch.tensor([[high + 4, 2, high + 8, high, 1], [high + 1, high + 6, -1, -1, -1]], dtype=torch.int32, device=gpu)
    mine = tables[tables >= 0].long()
    gen = torch.Generator(device=gpu).manual_seed(3)

    def fill(part):
        x = torch.randint(-30000, 30000, (len(mine), *part.shape[1:]), generator=gen, device=gpu).to(torch.int16)
        part.view(torch.uint8 if part.dtype == torch.uint8 else torch.int16)[mine] = x.to(torch.uint8) if bits == 4 and (
            part.dtype == torch.uint8) else x & 0x3FFF  # (finite numbers)
        return part

    if bits == 16:
        cache = tuple(fill(torch.empty(blocks, bs, kv, dim, dtype=torch.bfloat16, device=gpu)) for _ in range(2))
    else:
        cache = KVCache4(blocks, bs, kv, dim, gpu)
        for part in cache.parts:
            fill(part)

    def rows(r, n):
        """The first n tokens of request r: (k, v)"""
        slots = (tables[r].long()[:, None] * bs + torch.arange(bs, device=gpu)).flatten()[:n]
        if bits == 4:
            return read_kv4(cache, slots, torch.float32)
        return [c[slots // bs, slots % bs] for c in cache]

    weights = torch.rand(blocks, bs, generator=gen, device=gpu)
    lens_, budget_ = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in (lens, budget)]
    want = []
    for r in range(2):
        w = weights[tables[r].clamp(min=0).long()].flatten()[:lens[r]].tolist()
        stay = torch.tensor(W.stays(w, lens[r], budget[r], 5, 10), device=gpu)
        want.append(([x[stay] for x in rows(r, lens[r])], torch.tensor(w, device=gpu)[stay]))
    kept = evict_tokens(weights, lens_, budget_, tables, [cache], sinks=5, recent=10)
    assert kept.tolist() == budget
    for r in range(2):
        for x, y in zip(rows(r, budget[r]), want[r][0]):
            assert torch.equal(x, y)
        assert torch.equal(weights[tables[r].clamp(min=0).long()].flatten()[:budget[r]], want[r][1])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [1, 5, 90])
def test_sums_by_the_lse_of_rows_that_see_nothing(gpu, tokens, bits):
    """window_attention's lse as it is, -inf for rows all of whose tokens are absent"""
    b = Batch(tokens, [tokens + 40, tokens, 33, 3], [tokens, tokens, 1, 3 + tokens], 8, 2, 64, 16, torch.bfloat16, bits)
    b.tables[0, -2:], b.tables[1], b.tables[2, 1:] = -1, -1, 1 << 20
    args = b.args(gpu)
    for seen in ({"window": 12, "sinks": 0}, {"window": 30, "sinks": 2}, {"window": None, "sinks": 0}):
        _, lse = (window_attention4 if bits == 4 else window_attention)(*args, return_lse=True, **seen)
        given = lse.double().cpu().numpy()
        assert (given == -float("inf")).any()
        sums = torch.zeros(b.blocks, b.bs, device=gpu)
        accumulate_weights(args[0], args[1], *args[-3:], lse, sums, **seen)
        want, far = W.accumulate(sums.cpu().numpy() * 0, b.q.double().numpy(), b.dense()[0], b.tables, b.lens, b.offsets,
                                 given, b.dim ** -0.5, None, **seen)
        check_weights(b, sums, want, far)


@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_and_single_tokens_in_calls_of_their_own(gpu, bits):
    """Two calls over slices of one batch's requests, into one output and one tensor of sums"""
    tokens = [300, 70] + [1] * 9
    lens = [400, 70] + [1 + 37 * i for i in range(9)]
    b = Batch(2, lens, tokens, 16, 2, 128, 16, torch.bfloat16, bits, pad=3)
    q, *cache, tables, lens_, offsets = b.args(gpu)
    seen = {"window": 150, "sinks": 3}
    attend = window_attention4 if bits == 4 else window_attention
    out, whole = torch.full_like(q, 9.0), torch.full(q.shape[:2], float("nan"), device=gpu)
    sums = torch.zeros(b.blocks, b.bs, device=gpu)
    for part, most in ((slice(0, 2), 300), (slice(2, 11), 1)):
        some = (tables[part], lens_[part], offsets[part.start:part.stop + 1])
        _, lse = attend(q, *cache, *some, max_tokens=most, max_context=400, return_lse=True, out=out, **seen)
        rows = slice(b.offsets[part.start], b.offsets[part.stop])
        whole[rows] = lse[rows]
        accumulate_weights(q, cache[0], *some, lse, sums, max_tokens=most, max_context=400, **seen)
    assert (out[-3:] == 9.0).all()
    b.check((out, whole), b.oracle(**seen))
    want, far = W.accumulate(sums.cpu().numpy() * 0, b.q.double().numpy(), b.dense()[0], b.tables, b.lens, b.offsets,
                             torch.nan_to_num(whole).double().cpu().numpy(), b.dim ** -0.5, None, **seen)
    check_weights(b, sums, want, far)


def sums_of(b, args, lse, start, cache=None, **kw):
    """accumulate_weights on a copy of start, and the check of it against the oracle"""
    sums = start.clone()
    accumulate_weights(args[0], cache if cache is not None else args[1], *args[-3:], lse, sums, **kw)
    given = lse.double().cpu().numpy()
    if kw.get("max_tokens") is not None:
        for r in range(len(b.lens)):  # (rows beyond it: e^-10000)
            given[b.offsets[r] + kw["max_tokens"]:b.offsets[r + 1]] = 1e4
    scale = kw.get("scale")
    want, far = W.accumulate(start.cpu().numpy(), b.q[:len(given)].double().numpy(), b.dense()[0], b.tables, b.lens, b.offsets,
                             given, b.dim ** -0.5 if scale is None else scale, None, kw.get("window"), kw.get("sinks", 0))
    # check_weights' bound, and beside it 2^-126 for each of the weights that are added: fp32 has no normal
    # number below, and an exponential that is smaller may come as 0
    rows = b.offsets[-1] * b.heads
    e = (b.dim + 12) * 2.0 ** -23 * far + 2.0 ** -20 + (rows + 16) * 2.0 ** -24
    assert (np.abs(sums.double().cpu().numpy() - want) <= e * np.abs(want) + rows * 2.0 ** -126).all(), f"{kw}"
    return sums


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 20.0])
def test_sums_of_other_scales(gpu, scale, tokens, bits):
    b = Batch(tokens, [tokens + 90, 33, 70], [tokens, 1, min(tokens, 20)], 4, 2, 64, 16, torch.float16, bits)
    args, kw = b.args(gpu), {"window": 50, "sinks": 3, "scale": scale}
    _, lse = (window_attention4 if bits == 4 else window_attention)(*args, return_lse=True, **kw)
    sums_of(b, args, lse, torch.zeros(b.blocks, b.bs, device=gpu), **kw)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("bs", [32, 48, 80, 256])
@pytest.mark.parametrize("tokens", [1, 2, 30, 300])
@pytest.mark.parametrize("heads,kv,dim", [(16, 2, 128), (14, 2, 64)])
def test_sums_over_blocks_of_other_sizes_and_rows_beyond_max_tokens(gpu, heads, kv, dim, tokens, bs, bits):
    b = Batch(bs, [tokens + 500, 257, 40], [tokens, 1, min(tokens, 40)], heads, kv, dim, bs, torch.bfloat16, bits,
              garbage=float("nan"))
    args, start = b.args(gpu), torch.rand(b.blocks, bs, device=gpu)
    _, lse = (window_attention4 if bits == 4 else window_attention)(*args, return_lse=True, window=200, sinks=10)
    whole = sums_of(b, args, lse, start, window=200, sinks=10)
    assert torch.equal(whole, sums_of(b, args, lse, start, window=200, sinks=10, max_tokens=tokens))
    if tokens > 1:
        sums_of(b, args, lse, start, window=200, sinks=10, max_tokens=max(1, tokens - 3))


@pytest.mark.parametrize("tokens", [1, 60])
def test_sums_from_rows_and_keys_of_other_strides(gpu, tokens):
    b = Batch(6, [tokens + 300, 100], [tokens, min(tokens, 9)], 8, 2, 128, 16, torch.bfloat16)
    q, k, v, *rest = args = b.args(gpu)
    _, lse = window_attention(*args, return_lse=True)
    start = torch.zeros(b.blocks, b.bs, device=gpu)
    want = sums_of(b, args, lse, start)
    fused = torch.full((q.shape[0], 12, 128), float("nan"), dtype=q.dtype, device=gpu)
    fused[:, 2:10] = q
    turned = k.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((v, k), 3)[:, :, :, 1]
    far = torch.full((b.blocks, 3, b.bs, 2, 128), float("nan"), dtype=k.dtype, device=gpu)[:, 1]
    far.copy_(k)
    for rows in (q, fused[:, 2:10], q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)):
        for keys in (k, turned, both, far):
            assert torch.equal(sums_of(b, [rows, keys, *rest], lse, start), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("bs", [32, 48, 80, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_over_blocks_of_other_sizes(gpu, dtype, bs, bits):
    b = Batch(bs, [700, 257, 40, 128], [300, 1, 40, 0], 16, 2, 128, bs, dtype, bits, garbage=float("inf"))
    args = b.args(gpu)
    q = torch.nn.functional.pad(args[0], (0, 0, 0, 0, 0, 40000))  # (as many rows as make it one of many)
    attend, n = window_attention4 if bits == 4 else window_attention, b.offsets[-1]
    for window, sinks in ((None, 0), (130, 20), (64, 200), (1, 1)):
        out, lse = attend(q, *args[1:], window=window, sinks=sinks, return_lse=True)
        b.check((out[:n], lse[:n]), b.oracle(window=window, sinks=sinks), f"{window} {sinks}")
