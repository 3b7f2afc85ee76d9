"""Attention over a sliding window with sinks, the cache in 16 and in 4 bits, against the
oracle in 64 bits (tests/bounded.py: the bounds)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from pageserve_amd import KVCache4, tree_attention, window_attention, window_attention4, write_kv4
from bounded import HEADS, Batch

pytestmark = pytest.mark.gpu


def attend(b, gpu, args=None, **kw):
    return (window_attention4 if b.bits == 4 else window_attention)(*(args or b.args(gpu)), **kw)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 33, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
def test_lengths_windows_and_sinks(gpu, heads, tokens, dtype, bits):
    lens = [tokens, tokens + 1, 15, 16, 17, 33, 200, 300]
    rng = np.random.default_rng(tokens)
    counts = [tokens, tokens] + [min(int(n), x) for n, x in zip(rng.integers(0, tokens + 1, 4), lens[2:])] + [tokens, 0]
    b = Batch(tokens, lens, counts, *HEADS[heads], 16, dtype, bits, garbage=float("nan"))
    args = b.args(gpu)
    for window, sinks in ((None, 0), (1, 0), (20, 4), (64, 40), (500, 3)):
        want = b.oracle(window=window, sinks=sinks)
        kw = {"window": window, "sinks": sinks}
        b.check(attend(b, gpu, args, return_lse=True, **kw), want, f"{kw}")
        b.check(attend(b, gpu, args, max_tokens=tokens, max_context=300, **kw), want, f"{kw}, bounds given")
    # any expected context gives the same result to rounding: other splits
    for context in (0, 100, 5000, 10 ** 6):
        b.check(attend(b, gpu, args, max_context=context, return_lse=True, **kw), want, f"max_context={context}")


@pytest.mark.parametrize("lens,tokens,bs", [([1500, 3], [1, 1], 16), ([4000], [7], 48), ([2000, 0, 777], [40, 0, 3], 64),
                                            ([31, 32, 33, 64, 65], [1, 2, 1, 2, 1], 32), ([2049], [1], 256),
                                            ([700, 650], [300, 129], 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (130, 0), (600, 37)])
@pytest.mark.parametrize("bits", [16, 4])
def test_longer_contexts(gpu, lens, tokens, bs, window, sinks, bits):
    b = Batch(sum(lens), lens, tokens, 16, 2, 128, bs, torch.bfloat16, bits, garbage=float("inf"))
    b.check(attend(b, gpu, window=window, sinks=sinks, max_tokens=max(tokens), max_context=max(lens), return_lse=True),
            b.oracle(window=window, sinks=sinks))
