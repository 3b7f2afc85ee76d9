"""Pins of the drafting oracle (oracle/drafting_oracle.py) against hand-worked
values and exact rationals, and the CPU form of the 4-bit weights against it."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import drafting_oracle as D
from pageserve_amd import QuantizedWeight4
from pageserve_amd.quantization4 import VALUES


def _weights(seed, n, k):
    return (np.random.default_rng(seed).standard_normal((n, k)) * 0.02).astype(np.float32)


def test_the_nearest_value_is_taken_and_ties_go_to_the_even_code():
    w = _weights(1, 4, 64)
    w[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]  # scale 1: the midpoints
    w[0, 8:] = 0
    w[1, :32] = 0
    codes, scale = D.quantize4(w, 32)
    assert scale[0, 0] == 1.0 and codes[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]
    assert scale[1, 0] == D.bf16(np.float32(1e-8) / np.float32(6)) and not codes[1, :32].any()
    for r in range(2, 4):
        for j in range(64):
            s = Fraction(float(scale[r, j // 32]))
            far = [abs(abs(Fraction(float(w[r, j]))) - Fraction(v) * s) for v in D.VALUES.tolist()]
            best = min(range(8), key=lambda c: (far[c], c % 2))
            assert codes[r, j] % 8 == best and (codes[r, j] >= 8) == (w[r, j] < 0 and best > 0)
    assert list(VALUES) == D.VALUES.tolist()


@pytest.mark.parametrize("n,k,group", [(1, 16, 32), (3, 48, 32), (17, 144, 64), (16, 128, 128), (40, 272, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_cpu_weight_matches_the_oracle(n, k, group, dtype):
    w = torch.from_numpy(_weights(n + k, n, k)).to(dtype)
    codes, scale = D.quantize4(w.float().numpy(), group)
    qw = QuantizedWeight4(w, group)
    assert np.array_equal(qw.codes.numpy(), codes)
    assert np.array_equal(qw.scale.float().numpy(), scale) and qw.scale.dtype == torch.bfloat16
    want = torch.from_numpy(D.dense4(codes, scale, group)).to(dtype)
    assert torch.equal(qw.dense(), want) and qw.dense().dtype == dtype
    again = QuantizedWeight4.from_codes(qw.codes, qw.scale, group, dtype)
    assert torch.equal(again.qp, qw.qp) and torch.equal(again.sp.view(torch.int16), qw.sp.view(torch.int16))
    blocks = -(-n // 16) * -(-k // 128)
    assert qw.storage_bytes == blocks * (1024 + 32 * (128 // group))


@pytest.mark.parametrize("n,k", [(0, 64), (5, 0), (0, 0)])
def test_cpu_weight_without_rows_or_columns(n, k):
    qw = QuantizedWeight4(torch.zeros(n, k), 32)
    assert qw.codes.shape == qw.dense().shape == (n, k) and qw.scale.shape == (n, k // 32) and qw.storage_bytes == 0
    assert QuantizedWeight4.from_codes(qw.codes, qw.scale, 32).dense().shape == (n, k)


def test_not_finite_groups():
    w = _weights(5, 2, 64)
    w[0, 3], w[1, 40] = np.nan, np.inf
    codes, scale = D.quantize4(w, 32)
    qw = QuantizedWeight4(torch.from_numpy(w), 32)
    assert np.isnan(scale[0, 0]) and np.isinf(scale[1, 1]) and np.isfinite([scale[0, 1], scale[1, 0]]).all()
    assert np.array_equal(qw.codes.numpy(), codes) and np.array_equal(qw.scale.float().numpy(), scale, equal_nan=True)
    assert not codes[0, :32].any() and codes[1, 32:].astype(bool).sum() == 1


def test_a_parameter_leaves_no_graph():
    w = torch.nn.Parameter(torch.from_numpy(_weights(1, 20, 64)))
    qw = QuantizedWeight4(w, 32)
    again = QuantizedWeight4.from_codes(qw.codes, qw.scale.clone().requires_grad_(), 32, torch.float32)
    for t in (qw.qp, qw.sp, qw.scale, qw.dense(), again.sp, again.dense()):
        assert not t.requires_grad
    assert torch.equal(qw.dense(), again.dense())


@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.int32, torch.int64])
def test_codes_of_any_integer_type(dtype):
    """Torch's own arithmetic on masks and bytes yields int64: the same weight."""
    gen = torch.Generator().manual_seed(7)
    codes = torch.randint(0, 16, (20, 144), generator=gen, dtype=torch.uint8)
    scale = torch.rand(20, 5, generator=gen).bfloat16()
    want = QuantizedWeight4.from_codes(codes, scale, 32)
    got = QuantizedWeight4.from_codes(codes.to(dtype), scale, 32)
    assert torch.equal(got.qp, want.qp) and torch.equal(got.codes, codes)
    low = QuantizedWeight4.from_codes(codes.to(dtype) - 16, scale, 32)  # the low four bits count
    assert torch.equal(low.qp, want.qp)
    for bad in (codes.float(), codes.bool(), codes.to(torch.complex64)):
        with pytest.raises(TypeError, match="integer type"):
            QuantizedWeight4.from_codes(bad, scale, 32)
    with pytest.raises(TypeError, match="bf16"):
        QuantizedWeight4.from_codes(codes, scale.float(), 32)


def test_packed_layout():
    """Column 32 j + 8 g + i of row r of a block: bits 4 i of dword j of lane r + 16 g."""
    n, k, group = 20, 272, 32
    codes = np.random.default_rng(3).integers(0, 16, (n, k), dtype=np.uint8)
    scale = torch.randn(n, -(-k // group)).bfloat16()
    qw = QuantizedWeight4.from_codes(torch.from_numpy(codes), scale, group)
    words = qw.qp.numpy().view(np.uint32).reshape(-1, 64, 4)
    sp = qw.sp.view(2, 3, 16, 4)
    for r, c in [(0, 0), (5, 7), (15, 127), (16, 128), (19, 271), (3, 200)]:
        blk, kk = (r // 16) * 3 + c // 128, c % 128
        word = int(words[blk, r % 16 + 16 * (kk % 32 // 8), kk // 32])
        assert word >> (4 * (kk % 8)) & 15 == codes[r, c]
        assert sp[r // 16, c // 128, r % 16, kk // 32] == scale[r, c // 32]
    assert not words[5, :, 2:].any() and not (words[3:, 4:16].any())  # columns from 272 on, rows from 20 on


def test_append_and_truncate_by_hand():
    lens, tables = [3, 0, 4], [[7, -1, -1], [-1, -1, -1], [9, -1, -1]]
    free = [1, 2, 5, 6, 8]
    slots, status, count = D.append(lens, [2, 0, 5], [0, 2, 2, 7], tables, free, 5, 4, 8)
    assert status == [0, 0, 0] and lens == [5, 0, 9] and count == 2
    assert tables == [[7, 8, -1], [-1, -1, -1], [9, 6, 5]]
    assert slots == [31, 32, 24, 25, 26, 27, 20, -1]
    assert D.truncate(lens, [3, 0, 4], tables, free, count, 4) == 5
    assert lens == [3, 0, 4] and tables == [[7, -1, -1], [-1, -1, -1], [9, -1, -1]] and free == [1, 2, 5, 6, 8]
    # two blocks: the first request is served, the second not, the third needs none
    lens, tables = [4, 4, 2], [[0, -1, -1], [1, -1, -1], [2, -1, -1]]
    slots, status, count = D.append(lens, [8, 1, 1], [0, 1, 2, 3], tables, [3, 4], 2, 4, 3)
    assert status == [0, 1, 0] and lens == [12, 4, 3] and count == 0 and slots == [16, -1, 10]


def test_a_hole_in_a_table_is_not_given_back():
    lens, tables, free = [40, 20], [[3, -1, 5], [-1, 7, -1]], [9, 0, 0, 0, 0]
    count = D.truncate(lens, [0, 3], tables, free, 1, 16)
    assert count == 4 and free[:4] == [9, 7, 5, 3]
    assert lens == [0, 3] and tables == [[-1, -1, -1], [-1, -1, -1]]
    slots, status, count = D.append(lens, [40, 0], [0, 40, 40], tables, free, count, 16, 40)
    assert status == [0, 0] and count == 1 and tables[0] == [3, 5, 7] and min(slots) >= 0


def test_ancestors():
    assert D.ancestors([-1, 0, 0, 1, 5, 9]) == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {4}, {5}]
