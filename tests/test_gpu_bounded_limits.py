"""Calls of the operators of long texts whose grids pass what one launch may have: 2^32 threads."""

from __future__ import annotations

import pytest
import torch

from pageserve_amd import KVCache4, evict_tokens

pytestmark = pytest.mark.gpu


def numbers(gpu, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)


@pytest.mark.parametrize("bits,heads,dim", [(16, 8, 128), (4, 8, 64), (16, 16, 127), (16, 64, 128)])
def test_eviction_of_many_requests_in_many_layers(gpu, bits, heads, dim):
    """8192 requests x 8 heads x 16 layers and more: from 2^22 workgroups of 1024 threads on.  A few requests have tokens; the
    call gives what one of those alone gives."""
    requests, layers, bs, live, lens = 8192, 16, 16, [0, 1, 4095, 8190, 8191], [50, 16, 300, 47, 33]
    have = [-(-n // bs) for n in lens]
    blocks = sum(have) + 1
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    tables, all_lens = torch.full((requests, max(have)), -1, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    at = 0
    for b, n, h in zip(live, lens, have):
        tables[b, :h], all_lens[b] = order[at:at + h], n
        at += h
    budget = torch.full((requests,), 20, dtype=torch.int32)
    weights = numbers(gpu, blocks, bs, dtype=torch.float32)
    caches = []
    for i in range(layers):
        if bits == 16:
            caches.append(tuple(numbers(gpu, blocks, bs, heads, dim, seed=2 * i + j) for j in range(2)))
        else:
            c = KVCache4(blocks, bs, heads, dim, gpu)
            for j, p in enumerate(c.parts):
                p.copy_((numbers(gpu, *p.shape, dtype=torch.float32, seed=4 * i + j) * 1000).to(p.dtype))
            caches.append(c)

    def parts(caches):
        return [p for c in caches for p in (c.parts if bits == 4 else c)]

    def copy(caches):
        return [KVCache4.of(*(p.clone() for p in c.parts)) if bits == 4 else tuple(p.clone() for p in c) for c in caches]

    def call(rows, weights, caches):
        return evict_tokens(weights, all_lens[rows].to(gpu), budget[rows].to(gpu), tables[rows].to(gpu), caches, sinks=2, recent=3)

    want_weights, want = weights.clone(), copy(caches)
    before = copy(caches)
    assert call(live, want_weights, want).tolist() == [20, 16, 20, 20, 20]
    assert not all(torch.equal(x, y) for x, y in zip(parts(want), parts(before)))
    kept = call(list(range(requests)), weights, caches)
    assert torch.equal(kept.cpu(), torch.minimum(all_lens, budget))
    assert torch.equal(weights, want_weights)
    for x, y in zip(parts(caches), parts(want)):
        assert torch.equal(x, y)
