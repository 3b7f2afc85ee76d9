"""Rows into the 4-bit cache and back, against the oracle bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import window_oracle as W
from pageserve_amd import KVCache4, append_blocks, read_kv4, write_kv4

pytestmark = pytest.mark.gpu


def rows(seed, n, kv, dim, dtype, std=1.0):
    return (torch.from_numpy(np.random.default_rng(seed).standard_normal((n, kv, dim))) * std).to(dtype)


def dense(x):
    return W.dense_rows(*W.quantize_rows(x.to(torch.float32).numpy()))


def same(got, want):
    """float64 `want` exactly, NaN for NaN"""
    return np.array_equal(got.to(torch.float64).cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("kv,dim", [(2, 128), (2, 64), (1, 64), (3, 128), (7, 64)])
@pytest.mark.parametrize("n,bs", [(1, 16), (5, 16), (33, 48), (300, 64), (1000, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_come_back_as_the_oracle_rounds_them(gpu, kv, dim, n, bs, dtype):
    k, v = rows(n, n, kv, dim, dtype), rows(n + 1, n, kv, dim, dtype, 0.01)
    blocks = n // bs + 3
    slots = torch.from_numpy(np.random.default_rng(n).permutation(blocks * bs)[:n])
    c = KVCache4(blocks, bs, kv, dim, gpu)
    write_kv4(k.to(gpu), v.to(gpu), c, slots.to(gpu))
    for kind in (torch.float32, torch.bfloat16):
        gk, gv = read_kv4(c, slots.to(gpu), kind)
        assert gk.dtype == kind and gk.shape == (n, kv, dim)
        # (value * scale is a bf16 number: exact in both)
        assert same(gk, dense(k)) and same(gv, dense(v))
    gk, _ = read_kv4(c, slots.to(gpu), torch.float16)
    assert same(gk, dense(k))  # (8 bits, in fp16's range here)
    # the other slots are zeros still
    rest = torch.from_numpy(np.setdiff1d(np.arange(blocks * bs), slots.numpy())).to(gpu)
    assert not any(x.any() for x in read_kv4(c, rest))


@pytest.mark.parametrize("dim", [64, 128])
def test_the_layout_is_the_documented_one(gpu, dim):
    n, kv, bs = 40, 2, 16
    k, v = rows(1, n, kv, dim, torch.bfloat16), rows(2, n, kv, dim, torch.bfloat16)
    c = KVCache4(3, bs, kv, dim, gpu)
    write_kv4(k.to(gpu), v.to(gpu), c, torch.arange(n, device=gpu))
    (kq, ks), (vq, vs) = (W.quantize_rows(x.float().numpy()) for x in (k, v))
    C = dim // 32
    gk, gv = c.k.cpu().numpy(), c.v.cpu().numpy().reshape(3, kv, -1)
    for i in range(n):
        b, t = divmod(i, bs)
        for h in range(kv):
            for d in range(dim):
                byte = 4 * (C * (d % 32 // 8) + d // 32) + d % 8 // 2
                assert gk[b, h, t, byte] >> (4 * (d % 2)) & 15 == kq[i, h, d]
                m, at = d % 16, d // 16
                byte = t // 16 * 16 * (dim // 2) + C * (4 * (16 * (t % 16 // 4) + m) + t % 4) + at // 2
                assert gv[b, h, byte] >> (4 * (at % 2)) & 15 == vq[i, h, d]
            assert np.array_equal(c.k_scale[b, h, t].float().cpu().numpy(), ks[i, h])
            assert np.array_equal(c.v_scale[b, h, t].float().cpu().numpy(), vs[i, h])


def test_borders_zeros_tiny_and_large_numbers(gpu):
    x = torch.zeros(12, 1, 64, dtype=torch.bfloat16)
    x[0, 0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])  # scale 1: the midpoints
    x[1, 0, 32:40] = -torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[2] = -0.0
    x[3] = 1e-12
    x[4] = torch.finfo(torch.bfloat16).max
    x[5, 0, ::2] = -torch.finfo(torch.bfloat16).max
    x[6, 0, 3] = float("nan")
    x[7, 0, 40] = float("inf")
    x[8, 0, 40] = -float("inf")
    x[9, 0, 1], x[9, 0, 2] = float("inf"), float("nan")
    x[10] = torch.linspace(-7, 9, 64)
    x[11] = torch.finfo(torch.bfloat16).tiny
    for y in (x, x.clamp(-65504, 65504).to(torch.float16)):
        c = KVCache4(1, 16, 1, 64, gpu)
        slots = torch.arange(12, device=gpu)
        write_kv4(y.to(gpu), y.flip(2).contiguous().to(gpu), c, slots)
        gk, gv = read_kv4(c, slots, torch.float32)
        assert same(gk, dense(y)) and same(gv, dense(y.flip(2)))
        # nothing finite has become infinite in the rows' own type
        fine = torch.isfinite(y).view(12, 2, 32).all(2)
        got = read_kv4(c, slots, y.dtype)[0].cpu().view(12, 2, 32)
        assert torch.isfinite(got[fine]).all()


def test_slots_outside_and_rows_of_any_strides(gpu):
    kv, dim, bs = 2, 128, 16
    wide = rows(3, 50, 2 * kv, dim, torch.bfloat16).to(gpu)
    k, v = wide[:, ::2], wide[:, 1::2]
    slots = torch.tensor([-1, 0, 5, 48, 47, -7, 1 << 40] + list(range(6, 47)) + [2, 3], device=gpu)
    c = KVCache4(3, bs, kv, dim, gpu)
    write_kv4(k, v, c, slots)
    inside = ((slots >= 0) & (slots < 48)).cpu().numpy()
    gk, gv = read_kv4(c, slots, torch.float32)
    for g, x in ((gk, k), (gv, v)):
        want = np.where(inside[:, None, None], dense(x.cpu()), 0)
        assert same(g, want)
    # (permuted, shifted by an element, transposed dims)
    odd = torch.empty(51 * kv * dim + 1, dtype=torch.bfloat16, device=gpu)[1:50 * kv * dim + 1].view(50, kv, dim)
    odd.copy_(k)
    c2, c3 = KVCache4(3, bs, kv, dim, gpu), KVCache4(3, bs, kv, dim, gpu)
    write_kv4(odd, v.permute(1, 0, 2).contiguous().permute(1, 0, 2), c2, slots)
    write_kv4(k.transpose(1, 2).contiguous().transpose(1, 2), v, c3, slots)
    for p, p2, p3 in zip(c.parts, c2.parts, c3.parts):
        assert torch.equal(p.view(torch.uint8), p2.view(torch.uint8)) and torch.equal(p.view(torch.uint8), p3.view(torch.uint8))


def test_no_rows_and_an_empty_cache(gpu):
    c = KVCache4(0, 16, 2, 64, gpu)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    write_kv4(none, none, c, torch.empty(0, dtype=torch.long, device=gpu))
    k, v = read_kv4(c, torch.tensor([0, -1], device=gpu))
    assert k.shape == v.shape == (2, 2, 64) and not k.any()


def test_refusals(gpu):
    c = KVCache4(2, 16, 2, 64, gpu)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    s = torch.arange(3, device=gpu)
    with pytest.raises(TypeError):
        write_kv4(k.float(), k, c, s)
    with pytest.raises(TypeError):
        write_kv4(k, k.half(), c, s)
    with pytest.raises(TypeError):
        write_kv4(k, k, c, s.int())
    for bad in (k[:2], k[:, :1], k[:, :, :32], k[0]):
        with pytest.raises(ValueError):
            write_kv4(bad, k, c, s)
    with pytest.raises(ValueError):
        write_kv4(k, k.cpu(), c, s)
    with pytest.raises(RuntimeError):
        write_kv4(k, k, KVCache4(2, 16, 2, 64, "cpu"), s)
    with pytest.raises(ValueError):  # (codes of another shape than the scales)
        write_kv4(k, k, KVCache4.of(c.k, c.k_scale[:1].contiguous(), c.v, c.v_scale), s)
    with pytest.raises(ValueError):
        write_kv4(k, k, KVCache4.of(c.k.transpose(1, 2), c.k_scale, c.v, c.v_scale), s)
    with pytest.raises(TypeError):
        write_kv4(k, k, KVCache4.of(c.k, c.k_scale.float(), c.v, c.v_scale), s)
    with pytest.raises(TypeError):
        read_kv4(c, s, torch.float64)
    with pytest.raises(ValueError):
        read_kv4(c, s[::2])


def test_after_append_blocks_in_a_graph(gpu):
    """A prompt's rows and then single tokens, slots from append_blocks, captured and replayed."""
    kv, dim, bs, n = 2, 128, 16, 4
    i32 = dict(dtype=torch.int32, device=gpu)
    lens, tables = torch.zeros(n, **i32), torch.full((n, 8), -1, **i32)
    free, count = torch.arange(32, **i32), torch.tensor([32], **i32)
    c = KVCache4(32, bs, kv, dim, gpu)
    new, offsets = torch.tensor([30, 1, 0, 17], **i32), torch.tensor([0, 30, 31, 31, 48], **i32)
    x = rows(5, 48, kv, dim, torch.bfloat16).to(gpu)
    slots, status = append_blocks(lens, new, offsets, tables, free, count, bs, 48)
    write_kv4(x, -x, c, slots)
    one, step = torch.ones(n, **i32), torch.arange(n + 1, **i32)
    y = rows(6, n, kv, dim, torch.bfloat16).to(gpu)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        s, _ = append_blocks(lens, one, step, tables, free, count, bs, n)
        write_kv4(y, -y, c, s)
        gk, gv = read_kv4(c, s, torch.float32)
    for turn in range(5):
        y.copy_(rows(10 + turn, n, kv, dim, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = dense(y.cpu())
        assert same(gk, want) and same(gv, -want)
        assert lens.tolist() == [31 + turn, 2 + turn, 1 + turn, 18 + turn]
    # the prompt's rows are as they were written
    gk, gv = read_kv4(c, slots, torch.float32)
    assert same(gk, dense(x.cpu())) and not status.any()
