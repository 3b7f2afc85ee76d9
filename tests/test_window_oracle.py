"""Pins of the oracle of long texts (oracle/window_oracle.py) against hand-worked values,
exact rationals and torch, and refusals that need no GPU."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import window_oracle as W
from pageserve_amd import KVCache4, accumulate_weights, evict_tokens, read_kv4, window_attention, window_attention4, write_kv4


def test_which_tokens_a_row_sees():
    assert W.sees(2, 5).tolist() == [[1, 1, 1, 1, 0], [1, 1, 1, 1, 1]]
    assert W.sees(2, 5, window=2).tolist() == [[0, 0, 1, 1, 0], [0, 0, 0, 1, 1]]
    assert W.sees(2, 5, window=1, sinks=2).tolist() == [[1, 1, 0, 1, 0], [1, 1, 0, 0, 1]]
    # (sinks that reach into the window, and rows that stand before the text)
    assert W.sees(1, 4, window=2, sinks=9).tolist() == [[1, 1, 1, 1]]
    assert W.sees(3, 2, window=5).tolist() == [[0, 0], [1, 0], [1, 1]]


def test_scales_are_the_first_six_bits_and_codes_the_nearest():
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((20, 64)) * np.exp(rng.standard_normal((20, 1)) * 4)).astype(np.float32)
    x[0, :8] = [0.25, -0.75, 1.25, 1.75, -2.5, 3.5, 5.0, 6.0]  # scale 1: the midpoints
    x[0, 8:32] = 0
    codes, scale = W.quantize_rows(x)
    assert scale[0, 0] == 1.0 and codes[0, :8].tolist() == [0, 10, 2, 4, 12, 6, 6, 7]
    for r in range(20):
        for g in range(2):
            part = x[r, 32 * g:32 * g + 32]
            full = Fraction(float(np.float32(np.abs(part).max()) / np.float32(6)))
            s = Fraction(float(scale[r, g]))
            assert s <= full < s * Fraction(33, 32) and 6 * s <= Fraction(float(np.abs(part).max())) * Fraction(1000001, 1000000)
            m = s
            while m.denominator > 1:
                m *= 2
            while m % 2 == 0:
                m /= 2
            assert m < 64  # six bits
            for i, v in enumerate(part):
                far = [abs(abs(Fraction(float(v))) - Fraction(float(u)) * s) for u in W.VALUES]
                best = min(range(8), key=lambda c: (far[c], c % 2))
                assert codes[r, 32 * g + i] == best + 8 * (v < 0 and best > 0)
    # value * scale is a bf16 number
    dense = torch.from_numpy(W.dense_rows(codes, scale))
    assert torch.equal(dense.to(torch.bfloat16).double(), dense)


def _attention_case(seed, n, length, window, sinks):
    rng = np.random.default_rng(seed)
    q, k, v = rng.standard_normal((n, 2, 8)), rng.standard_normal((length, 1, 8)), rng.standard_normal((length, 1, 8))
    mask = torch.from_numpy(W.sees(n, length, window, sinks))
    want = torch.nn.functional.scaled_dot_product_attention(
        torch.from_numpy(q).transpose(0, 1), torch.from_numpy(k).transpose(0, 1).expand(2, -1, -1),
        torch.from_numpy(v).transpose(0, 1).expand(2, -1, -1), mask, scale=0.5).transpose(0, 1).numpy()
    return q, k, v, want


@pytest.mark.parametrize("n,length,window,sinks", [(1, 1, None, 0), (4, 9, None, 0), (4, 9, 3, 0), (4, 20, 3, 2), (9, 9, 2, 1)])
def test_attention_against_torch(n, length, window, sinks):
    q, k, v, want = _attention_case(n + length, n, length, window, sinks)
    bs = 4
    blocks = -(-length // bs)
    kc, vc = (np.full((blocks + 1, bs, 1, 8), np.nan) for _ in range(2))
    table = np.random.default_rng(1).permutation(blocks + 1)[:blocks]
    for j in range(length):
        kc[table[j // bs], j % bs], vc[table[j // bs], j % bs] = k[j], v[j]
    out, lse, spread, mass, reach = W.attention(q, kc, vc, [table], [length], [0, n], 0.5, window, sinks)
    assert np.allclose(out, want, atol=1e-12) and (spread >= mass).all() and (reach > 0).all()
    see = W.sees(n, length, window, sinks)
    s = np.where(see[:, None], np.einsum("thd,jd->thj", q, k[:, 0]) * 0.5, -np.inf)
    assert np.allclose(lse, np.log(np.exp(s).sum(-1)))
    # the weights of a token: what its column of the softmax adds up to, new tokens from nothing
    start = np.arange((blocks + 1) * bs, dtype=np.float64).reshape(-1, bs)
    got, _ = W.accumulate(start, q, kc, [table], [length], [0, n], lse, 0.5, [n], window, sinks)
    p = np.exp(s - lse[..., None]).sum((0, 1))
    for j in range(length):
        old = 0 if j >= length - n else start[table[j // bs], j % bs]
        assert np.isclose(got[table[j // bs], j % bs], old + p[j])


def test_planted_mistakes_are_seen():
    """A window off by one, sinks left out and rows off by one change the result by far more
    than any bound of the tests."""
    q, k, v, want = _attention_case(3, 4, 30, 6, 2)
    for other in ((5, 2), (7, 2), (6, 0), (6, 1), (6, 3)):
        _, _, _, wrong = _attention_case(3, 4, 30, *other)
        assert np.abs(wrong - want).max() > 0.05


def test_what_stays():
    w = [5, 1, 9, 1, 7, float("nan"), 3, None]
    assert W.stays(w, 8, 8) == list(range(8)) and W.stays(w, 8, 99) == list(range(8)) and W.stays(w, 8, -1) == []
    assert W.stays(w, 8, 3) == [2, 4, 5]
    assert W.stays(w, 8, 6) == [0, 1, 2, 4, 5, 6]  # (of equal ones the first; an absent one last)
    assert W.stays(w, 8, 4, sinks=2, recent=1) == [0, 1, 5, 7]
    assert W.stays(w, 8, 3, sinks=2, recent=9) == [0, 1, 7] and W.stays(w, 8, 2, sinks=5, recent=9) == [0, 1]
    weights, cache = np.float32([[5, 1, 9, 1]]), np.arange(4.0).reshape(1, 4, 1)
    assert W.evict(weights, [[0]], [4], [2], [cache]) == [2]
    assert weights.tolist() == [[5, 9, 9, 1]] and cache.ravel().tolist() == [0, 2, 2, 3]
    assert W.evict(weights, [[0]], [4], [2], [cache], max_context=3) == [4]


def test_cpu_tensors_are_refused():
    c = KVCache4(2, 16, 2, 64, "cpu")
    rows, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)
    ints = torch.zeros(2, dtype=torch.int32)
    table, cache = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: write_kv4(rows, rows, c, slots), lambda: read_kv4(c, slots),
                 lambda: window_attention(rows, cache, cache, table, ints[:1], ints),
                 lambda: window_attention4(rows, c, table, ints[:1], ints),
                 lambda: accumulate_weights(rows, cache, table, ints[:1], ints, torch.zeros(3, 2), torch.zeros(2, 16)),
                 lambda: evict_tokens(torch.zeros(2, 16), ints[:1], ints[:1], table, [])):
        with pytest.raises(RuntimeError):
            call()


def test_a_caches_sizes():
    c = KVCache4(3, 32, 2, 128, "cpu")
    assert c.k.shape == c.v.shape == (3, 2, 32, 64) and c.k_scale.shape == c.v_scale.shape == (3, 2, 32, 4)
    assert c.storage_bytes == 3 * 32 * 2 * 2 * (64 + 8) and c.device == torch.device("cpu")
    assert KVCache4.of(*c.parts).parts == c.parts
    for bad in ({"head_dim": 96}, {"block_size": 24}, {"block_size": 0}):
        with pytest.raises(ValueError):
            KVCache4(**({"blocks": 3, "block_size": 32, "kv_heads": 2, "head_dim": 128, "device": "cpu"} | bad))
