"""A drafting step as it is used: 4-bit projections, attention of drafted trees over the
paged cache, and the accepted tokens appended and written, layer by layer.

Each operator is checked against its 64-bit form on the values that the GPU handed it
(the tolerances are those of the operators' own tests), and what the cache holds in
the end against the rows that were accepted, bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafting_oracle as D
from pageserve_amd import QuantizedWeight4, append_blocks, linear4, tree_attention, truncate_blocks, write_kv
from test_gpu_attend import Batch
from test_gpu_linear4 import _check

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, BS, LAYERS, GROUP = 192, 6, 2, 64, 16, 2, 64
REQUESTS, COLUMNS, TOKENS = 4, 8, 6


class Model:
    """Two layers with 4-bit weights and their caches; a batch of up to REQUESTS x TOKENS rows."""

    def __init__(self, gpu):
        rng = np.random.default_rng(5)
        self.gpu, self.dense, self.quant = gpu, [], []
        for layer in range(LAYERS):
            for n, k in (((HEADS + 2 * KV) * DIM, HIDDEN), (HIDDEN, HEADS * DIM)):
                codes, scale = D.quantize4((rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32), GROUP)
                self.dense.append(D.dense4(codes, scale, GROUP))
                self.quant.append(QuantizedWeight4.from_codes(torch.from_numpy(codes).to(gpu),
                                                              torch.from_numpy(scale).bfloat16().to(gpu), GROUP))
        blocks = REQUESTS * COLUMNS
        self.caches = [torch.zeros(2, blocks, BS, KV, DIM, dtype=torch.bfloat16, device=gpu) for _ in range(LAYERS)]
        i = dict(dtype=torch.int32, device=gpu)
        self.lens = torch.zeros(REQUESTS, **i)
        self.tables = torch.full((REQUESTS, COLUMNS), -1, **i)
        self.free = torch.as_tensor(rng.permutation(blocks), **i)
        self.count = torch.full((1,), blocks, **i)
        # the batch of a step
        rows = REQUESTS * TOKENS
        self.x = torch.zeros(rows, HIDDEN, dtype=torch.bfloat16, device=gpu)
        self.offsets = torch.zeros(REQUESTS + 1, **i)
        self.parents = torch.zeros(rows, **i)
        self.new = torch.zeros(REQUESTS, **i)
        self.index = torch.zeros(rows, **i)

    def step(self, seen=None):
        """The whole step, on the tensors above; (output rows, status)."""
        x, kvs = self.x, []
        for layer, (kc, vc) in enumerate(self.caches):
            qkv = linear4(x, self.quant[2 * layer]).view(-1, HEADS + 2 * KV, DIM)
            q, k, v = qkv.split([HEADS, KV, KV], 1)
            o = tree_attention(q, k, v, kc, vc, self.tables, self.lens, self.offsets, self.parents, max_tokens=TOKENS,
                               max_context=COLUMNS * BS)
            y = linear4(o.view(-1, HEADS * DIM), self.quant[2 * layer + 1], residual=x)
            if seen is not None:
                seen.append((x, qkv, o, y, kc.clone(), vc.clone()))
            kvs.append((k, v))
            x = y
        slots, status = append_blocks(self.lens, self.new, self.offsets, self.tables, self.free, self.count, BS,
                                      x.shape[0], self.index)
        for (k, v), (kc, vc) in zip(kvs, self.caches):
            write_kv(k, v, kc, vc, slots)
        return x, status

    def load(self, seed, tokens):
        """Random rows and trees of `tokens` per request; a path of each tree is accepted."""
        rng = np.random.default_rng(seed)
        rows, total = self.x.shape[0], sum(tokens)
        self.x.copy_(torch.from_numpy(rng.standard_normal((rows, HIDDEN))).bfloat16())
        offsets = np.concatenate([[0], np.cumsum(tokens)])
        parents, index, new = np.full(rows, -1), np.full(rows, -1), []
        for b, t in enumerate(tokens):
            for j in range(1, t):
                parents[offsets[b] + j] = rng.integers(max(j - 2, 0), j)
            path, j = [], int(rng.integers(0, t)) if t else -1
            while j >= 0:
                path.append(j)
                j = int(parents[offsets[b] + j])
            for n, j in enumerate(reversed(path)):
                index[offsets[b] + j] = n
            new.append(len(path))
        for dst, src in ((self.offsets, offsets), (self.parents, parents), (self.index, index), (self.new, new)):
            dst.copy_(torch.as_tensor(np.asarray(src), dtype=torch.int32))
        return offsets, parents, index, total

    def cached(self, layer, b):
        n = int(self.lens[b])
        blocks = self.tables[b, :-(-n // BS)].long()
        return self.caches[layer][:, blocks].flatten(1, 2)[:, :n]


def _attention(b, m, qkv, o, kc, vc, lens, tables, total, what):
    """o against the oracle on the rows that belong to a request."""
    probe = Batch.__new__(Batch)
    probe.lens, probe.dim, probe.dtype = lens, DIM, torch.bfloat16
    f = lambda t: t.to(torch.float64).cpu().numpy()  # noqa: E731
    q, k, v = (f(t) for t in qkv.split([HEADS, KV, KV], 1))
    want = D.tree_attention(q, k, v, f(kc), f(vc), tables, lens, b[0].tolist(), b[1].tolist(), DIM ** -0.5)
    probe.check(torch.cat([o[:total], o.new_zeros(o.shape[0] - total, HEADS, DIM)]), want, what)


STEPS = [[1, 6, 3, 0], [6, 6, 6, 6], [2, 0, 1, 5], [6, 1, 6, 6], [1, 1, 1, 1]]


def test_steps_against_the_oracle(gpu):
    m = Model(gpu)
    kept = [[[] for _ in range(REQUESTS)] for _ in range(LAYERS)]
    for turn, tokens in enumerate(STEPS * 2):
        b = m.load(turn, tokens)
        lens, tables, total = m.lens.tolist(), m.tables.cpu().numpy(), b[3]
        seen = []
        y, status = m.step(seen)
        assert status.tolist() == [0] * REQUESTS
        for layer, (x, qkv, o, out, kc, vc) in enumerate(seen):
            what = f"step {turn} layer {layer}"
            x64, o64 = (t[:total].to(torch.float64).cpu().numpy() for t in (x, o.flatten(1)))
            _check(qkv.flatten(1)[:total], m.dense[2 * layer], x64, GROUP, torch.bfloat16, what=what + " qkv")
            _attention(b, m, qkv, o, kc, vc, lens, tables, total, what)
            _check(out[:total], m.dense[2 * layer + 1], o64, GROUP, torch.bfloat16, residual=x64, what=what + " out")
            for r in range(REQUESTS):
                rows = [i for i in range(b[0][r], b[0][r + 1]) if b[2][i] >= 0]
                rows.sort(key=lambda i: b[2][i])
                kept[layer][r] += [qkv[i, HEADS:].clone() for i in rows]
                got = m.cached(layer, r)
                assert len(kept[layer][r]) == int(m.lens[r]) == got.shape[1]
                if rows:
                    want = torch.stack(kept[layer][r]).view(-1, 2, KV, DIM).transpose(0, 1)
                    assert torch.equal(got, want), what
    used = sum(-(-n // BS) for n in m.lens.tolist())
    assert int(m.count) == REQUESTS * COLUMNS - used
    # one request goes back to 3 tokens, one ends: what stays is untouched
    keep = m.lens.clone()
    keep[0], keep[1] = 3, 0
    truncate_blocks(m.lens, keep, m.tables, m.free, m.count, BS)
    assert m.lens.tolist() == keep.tolist() and int(m.count) == REQUESTS * COLUMNS - sum(
        -(-n // BS) for n in keep.tolist())
    held = m.tables[m.tables >= 0].tolist() + m.free[:int(m.count)].tolist()
    assert sorted(held) == list(range(REQUESTS * COLUMNS))
    for r in (0, 2, 3):
        want = torch.stack(kept[0][r][:int(m.lens[r])]).view(-1, 2, KV, DIM).transpose(0, 1)
        assert torch.equal(m.cached(0, r), want)


def test_an_accepted_path_reads_the_same_from_the_cache(gpu):
    """A token that follows a drafted path sees the same text when the path is in the cache."""
    m = Model(gpu)
    m.load(1, [6, 6, 6, 6])
    m.step()
    qkv = torch.randn(6, HEADS + 2 * KV, DIM, device=gpu).bfloat16()
    q, k, v = qkv.split([HEADS, KV, KV], 1)
    kc, vc = m.caches[0]
    i = dict(dtype=torch.int32, device=gpu)
    parents = torch.tensor([-1, 0, 0, 2, 1, 4], **i)  # the path 0, 1, 4, 5
    one = lambda n: torch.tensor([0, n], **i)  # noqa: E731
    lens, tables = m.lens[:1].clone(), m.tables[:1].clone()
    drafted = tree_attention(q, k, v, kc, vc, tables, lens, one(6), parents)
    index = torch.tensor([0, 1, -1, -1, 2, 3], **i)
    slots, status = append_blocks(lens, torch.tensor([3], **i), one(6), tables, m.free, m.count, BS, 6, index)
    assert status.tolist() == [0] and slots.tolist().count(-1) == 3
    write_kv(k, v, kc, vc, slots)
    args = (q[5:], k[5:], v[5:], kc, vc, tables, lens, one(1))
    cached = tree_attention(*args)
    f = lambda t: t.to(torch.float64).cpu().numpy()  # noqa: E731
    want = D.tree_attention(*(f(t) for t in args[:5]), tables.cpu().numpy(), lens.tolist(), [0, 1], None, DIM ** -0.5)
    probe = Batch.__new__(Batch)
    probe.lens, probe.dim, probe.dtype = lens.tolist(), DIM, torch.bfloat16
    probe.check(cached, want, "from the cache")
    probe.check(drafted[5:], want, "drafted")


def test_a_captured_step_replays(gpu):
    """The whole step in one graph, lengths, trees and tables changing between replays."""
    a, b = Model(gpu), Model(gpu)
    a.load(0, STEPS[0])
    a.step()
    a = Model(gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, status = a.step()
    for turn, tokens in enumerate(STEPS):
        a.load(turn, tokens)
        total = b.load(turn, tokens)[3]
        g.replay()
        want, ok = b.step()
        torch.cuda.synchronize()
        assert torch.equal(y[:total], want[:total]) and torch.equal(status, ok)
        assert torch.equal(a.lens, b.lens) and torch.equal(a.tables, b.tables) and torch.equal(a.count, b.count)
        assert all(torch.equal(p, q) for p, q in zip(a.caches, b.caches))
