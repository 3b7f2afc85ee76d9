"""Values that are not finite, in tiles of which a row group's first rows see a part and its last ones
all (or the other way round): each row that sees one has it in its output, whatever the other rows
of its workgroup see (tests/bounded.py: the bounds)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bounded import Batch
from oracle import window_oracle as W
from pageserve_amd import KVCache4, window_attention, window_attention4, write_kv4

pytestmark = pytest.mark.gpu

PAD = 40000  # rows of no request, as many as make the batch one of many rows


@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 64), (16, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 0), (300, 90), (7, 200)])
@pytest.mark.parametrize("first", [0, 13, 40, 1000])  # where row 0 stands
@pytest.mark.parametrize("bits,dtype", [(16, torch.bfloat16), (16, torch.float16), (4, torch.bfloat16), (4, torch.float16)])
@pytest.mark.parametrize("many", [True, False])
def test_values_that_are_not_finite_reach_all_rows_that_see_them(gpu, many, bits, dtype, first, window, sinks, heads, kv, dim):
    tokens = 90
    b = Batch(first, [first + tokens], [tokens], heads, kv, dim, 16, dtype, bits)
    q, *_, tables, lens, offsets = b.args(gpu)
    if many:
        q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, PAD))
    kc, vc = b.kc.to(gpu), b.vc.to(gpu)
    cache4 = KVCache4(b.blocks, 16, kv, dim, gpu) if bits == 4 else None
    slots = torch.arange(b.blocks * 16, device=gpu)

    def attend():
        kw = {"window": window, "sinks": sinks, "return_lse": True}
        if bits == 4:
            write_kv4(kc.flatten(0, 1), vc.flatten(0, 1), cache4, slots)
            out, lse = window_attention4(q, cache4, tables, lens, offsets, **kw)
        else:
            out, lse = window_attention(q, kc, vc, tables, lens, offsets, **kw)
        return out[:tokens], lse[:tokens]

    clean, lse = attend()
    want = b.oracle(window=window, sinks=sinks)
    b.check((clean, lse), want)
    see = torch.from_numpy(W.sees(tokens, first + tokens, window, sinks)).to(gpu)
    length, rows = first + tokens, slice((kv - 1) * (heads // kv), heads)  # (the rows of the last key head)
    near = sorted({j for j in [*range(first - 110, length, 7), first - 64, first, 0, 1, 63, 64, 127, 128, 191, length - 1]
                   if 0 <= j < length})
    for i, j in enumerate(near):
        at, value, d = (b.tables[0, j // 16], j % 16, kv - 1), (np.inf, -np.inf, np.nan)[i % 3], 37 * i % dim
        kept = vc[at].clone()
        vc[at + (d,)] = value
        out, got_lse = attend()
        vc[at] = kept
        hit = torch.zeros(out.shape, dtype=torch.bool, device=gpu)
        hit[:, rows, d] = see[:, j, None]
        there = out[hit].double()
        if bits == 4 or np.isnan(value):  # (an infinity in 4 bits is the scale of its 32 dims, zeros among them)
            assert not there.isfinite().any(), f"token {j}: rows that see it"
            if bits == 4:
                hit[:, rows, d // 32 * 32:d // 32 * 32 + 32] |= see[:, j, None, None]
        else:
            assert (there == value).all(), f"token {j}: rows that see it"
        b.check((torch.where(hit, clean, out), got_lse), want, f"token {j}")
