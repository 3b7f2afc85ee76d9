"""Tree attention over the paged cache against the oracle in 64 bits.

Tolerance per output.  A score is a sum of D exact products, each addition off by at
most 2^-23 of the magnitudes, then scaled: off by (D + 4) 2^-23 reach, reach = scale
max sum |q||k|.  So a weight p = 2^(score - m) is off by a factor of 1 + e, e = (D + 8)
2^-23 reach + 2^-20 (its own exponent's rounding lies in reach; v_exp_f32 and the
rescaling by a few more units), and its rounding to the type t by u = half a step of
t; a p that fp16 rounds to a multiple of 2^-24 may be off by 2^-25 instead, times at most
`keys` of them against a sum of at least 1.  out = sum p v / sum p with the same rounded
p above and below: off by (u + e) sum w (|v| + |out|), and a few fp32 additions in each of
keys / 32 steps, (keys / 32 + 64) 2^-23 of that sum; then the output's own rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafting_oracle as D
from pageserve_amd import tree_attention

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Batch:
    """A batch of requests on the CPU in float64-representable values of a type."""

    def __init__(self, seed, lens, tokens, heads, kv, dim, bs, dtype, parents="tree", pad=0, columns=None):
        rng = np.random.default_rng(seed)
        self.heads, self.kv, self.dim, self.bs, self.dtype = heads, kv, dim, bs, dtype
        self.lens, self.offsets = list(lens), np.concatenate([[0], np.cumsum(tokens)]).astype(int).tolist()
        rows = self.offsets[-1] + pad

        def values(*shape):
            return torch.from_numpy(rng.standard_normal(shape)).to(dtype)

        self.q, self.k, self.v = values(rows, heads, dim), values(rows, kv, dim), values(rows, kv, dim)
        have = [-(-n // bs) for n in lens]
        blocks = sum(have) + 2
        self.kc, self.vc = values(blocks, bs, kv, dim), values(blocks, bs, kv, dim)
        order, at = rng.permutation(blocks).tolist(), 0
        columns = columns if columns is not None else max(have)
        self.tables = np.full((len(have), columns), -1, dtype=np.int32)
        for b, h in enumerate(have):
            self.tables[b, :h] = order[at:at + h]
            at += h
        self.parents = None
        if parents == "tree":
            local = np.concatenate([np.arange(t) for t in tokens] + [np.zeros(pad)]).astype(int)
            self.parents = np.maximum(local - 1 - (rng.random(rows) ** 2 * 5).astype(int), -1)
        elif parents == "roots":
            self.parents = np.full(rows, -1)

    def oracle(self, scale=None, max_tokens=64):
        f = lambda t: t.to(torch.float64).numpy()  # noqa: E731
        return D.tree_attention(f(self.q), f(self.k), f(self.v), f(self.kc), f(self.vc), self.tables, self.lens,
                                self.offsets, None if self.parents is None else self.parents.tolist(),
                                self.dim ** -0.5 if scale is None else scale, max_tokens)

    def args(self, gpu):
        i = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(gpu)  # noqa: E731
        return [t.to(gpu) for t in (self.q, self.k, self.v, self.kc, self.vc)] + [
            i(self.tables), i(self.lens), i(self.offsets), None if self.parents is None else i(self.parents)]

    def check(self, got, want, what=""):
        out, spread, reach = want
        got = got.to(torch.float64).cpu().numpy()
        live = ~np.isnan(out)
        keys = max(list(self.lens) + [0]) + 64
        u = U[self.dtype]
        e = (self.dim + 8) * 2.0 ** -23 * reach[..., None] + 2.0 ** -20 + (keys / 32 + 64) * 2.0 ** -23
        if self.dtype is torch.float16:
            e = e + keys * 2.0 ** -25
        tol = (u + e) * spread
        tol = tol + u * (np.abs(out) + tol) + 2.0 ** -25
        off = np.where(live, np.abs(got - out) - tol, -1)
        assert not np.isnan(off).any(), f"{what}: not a number"
        assert (off <= 0).all(), f"{what}: {off.max():.3g} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


HEADS = {"3b": (16, 2, 128), "0.5b": (14, 2, 64), "one": (1, 1, 64), "each": (4, 4, 128), "wide": (24, 1, 128),
         "odd": (15, 3, 64)}


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 31, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths_and_trees(gpu, heads, tokens, dtype):
    lens = [0, 1, 15, 16, 17, 33, 200]
    rng = np.random.default_rng(tokens)
    counts = [tokens] + rng.integers(0, tokens + 1, len(lens) - 2).tolist() + [tokens]
    b = Batch(tokens, lens, counts, *HEADS[heads], 16, dtype)
    want = b.oracle()
    b.check(tree_attention(*b.args(gpu), max_tokens=tokens), want, "max_tokens given")
    b.check(tree_attention(*b.args(gpu)), want, "defaults")
    # any expected context gives the same result to rounding: other splits
    for context in (0, 100, 5000, 10 ** 6):
        b.check(tree_attention(*b.args(gpu), max_context=context, max_tokens=tokens), want, f"max_context={context}")


@pytest.mark.parametrize("lens,tokens,bs", [([1500, 3], [1, 1], 16), ([4000], [7], 48), ([2000, 0, 777], [40, 64, 3], 64),
                                            ([31, 32, 33, 64, 65], [1, 2, 1, 2, 1], 32), ([2049], [1], 256)])
@pytest.mark.parametrize("parents", ["tree", "chain", "roots"])
def test_longer_contexts(gpu, lens, tokens, bs, parents):
    b = Batch(sum(lens), lens, tokens, 16, 2, 128, bs, torch.bfloat16, parents)
    b.check(tree_attention(*b.args(gpu), max_tokens=max(tokens), max_context=max(lens)), b.oracle())


def test_scales_and_sharp_maxima(gpu):
    b = Batch(4, [300, 90], [9, 20], 14, 2, 64, 16, torch.bfloat16)
    for scale in (0.0, -0.3, 1.0, 4.0):
        b.check(tree_attention(*b.args(gpu), scale=scale), b.oracle(scale), f"scale={scale}")
    # scores that rise all along, and one key far above the rest, late
    b.kc *= torch.linspace(0.1, 3, b.kc.shape[0])[:, None, None, None].to(b.dtype)
    b.k[:, :, :] *= 4
    b.check(tree_attention(*b.args(gpu)), b.oracle(), "rising")


# kernels: few rows in one part and in many, 33 rows and more through LDS, one key slice and two
LARGE = [("0.5b", [300, 0], [1, 1], 1), ("3b", [5000], [1], 1), ("3b", [700, 40], [4, 3], 4), ("0.5b", [200], [9], 9),
         ("odd", [130, 260], [40, 64], 64), ("wide", [1000], [12], 12), ("3b", [257], [32], 32)]


@pytest.mark.parametrize("heads,lens,tokens,most", LARGE)
@pytest.mark.parametrize("dtype,powers", [(torch.float16, (3, 10, 12, 13)), (torch.bfloat16, (3, 10, 13, 30, 58))])
def test_large_scores_of_one_key(gpu, heads, lens, tokens, most, dtype, powers):
    """One key far above the rest, whose values are the answer, with nothing to round: a
    weight of 1 (to a factor near 1 that the sum has too) against zeros.  Scores of both
    signs from 2^6 or so to the type's largest, the key cached, first, last or among the others, or
    the token's own; a key that is there twice takes the mean, off by its rounding."""
    h, kv, dim = HEADS[heads]
    b = Batch(50, lens, tokens, h, kv, dim, 16, dtype, parents="roots")
    rng = np.random.default_rng(9)
    base = (torch.from_numpy(rng.uniform(0.5, 0.9, (kv, dim))) * torch.from_numpy(rng.choice([-1, 1], (kv, dim)))).to(dtype)
    b.k.zero_(), b.kc.zero_()
    rows = b.offsets[-1]
    for power in powers:
        # (a quarter of a power less for each further head: the scores differ and stay in range)
        size = [2.0 ** (power - i % 3) for i in range(h)]
        for sign in (1, -1):
            q = torch.stack([base[i // (h // kv)] * size[i] for i in range(h)])
            b.q[:] = q
            top = base * 2.0 ** power
            # sign 1: the key among zeros; -1: all others at twice the negative score
            rest = torch.zeros_like(top) if sign > 0 else -2 * top
            b.k[:], b.kc[:] = rest, rest
            want = torch.empty(rows, kv, dim, dtype=dtype)
            for r, n in enumerate(lens):
                lo, hi = b.offsets[r], b.offsets[r + 1]
                places = [0, n - 1, n // 2, n // 3] if n else []
                for t in range(lo, hi):
                    # the key in the cache (one place for the request), or the token itself
                    own = not places or r % 2
                    if own:
                        b.k[t] = sign * top
                        want[t] = b.v[t]
                if places and not r % 2:
                    at = places[(power + sign) % 4]
                    slot = int(b.tables[r, at // 16]), at % 16
                    b.kc[slot] = sign * top
                    want[lo:hi] = b.vc[slot]
            full = want.repeat_interleave(h // kv, 1)
            args = b.args(gpu)
            for kw in (dict(max_tokens=most), dict(max_tokens=most, max_context=1 << 20), dict()):
                got = tree_attention(*args, **kw).cpu()
                assert torch.equal(got, full), (power, sign, kw, (got.float() - full.float()).abs().max())
            # negative scale: the same scores from turned queries
            args[0] = -args[0]
            assert torch.equal(tree_attention(*args, max_tokens=most, scale=-(dim ** -0.5)).cpu(), full), (power, sign)
            if lens[0] > 32 and sign > 0:
                at = 20
                slot = int(b.tables[0, at // 16]), at % 16
                once = b.kc[slot].clone()
                b.kc[slot] = top
                if not torch.equal(once, top):
                    hi = b.offsets[1]
                    mean = (want[:hi].double() + b.vc[slot].double()) / 2
                    got = tree_attention(*b.args(gpu), max_tokens=most)[:hi].cpu().double()
                    mean = mean.repeat_interleave(h // kv, 1)
                    assert ((got - mean).abs() <= U[dtype] * mean.abs() + 2.0 ** -22).all(), (power, "twice")


@pytest.mark.parametrize("heads,requests,tokens", [("one", 1100, 1), ("one", 300, 33), ("3b", 140, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_small_weights_beside_a_large_one(gpu, heads, requests, tokens, dtype):
    """A first key at score 0 whose values are 0, 16383 more at 2^-x of its weight with
    values 1: out = n 2^-x / (1 + n 2^-x).  Weights are rounded by half a step of the type, u,
    fp16's no finer than 2^-32 of the largest; sums, exponents and the reciprocal by 2^-12 at most
    (16384 / 32 steps of 2^-23, and scores of at most 2^5 off by (D + 8) 2^-23 of that)."""
    h, kv, dim = HEADS[heads]
    n, bs = 16384, 64
    i = dict(dtype=torch.int32, device=gpu)
    tables = torch.arange(n // bs, **i).expand(requests, -1).contiguous()  # all read the same blocks
    rows = requests * tokens
    q = torch.zeros(rows, h, dim, dtype=dtype, device=gpu)
    q[..., 0] = 1
    kc, vc = (torch.zeros(n // bs, bs, kv, dim, dtype=dtype, device=gpu) for _ in range(2))
    k, v = (torch.zeros(rows, kv, dim, dtype=dtype, device=gpu) for _ in range(2))
    vc[:] = 1
    vc[0, 0] = 0
    offsets, lens = torch.arange(0, rows + 1, tokens, **i), torch.full((requests,), n, **i)
    k[..., 0] = -60000.0  # (the drafted tokens: nothing)
    for x in (20.5, 25.5, 27.25):
        kc[..., 0] = -x
        kc[0, 0, :, 0] = 0
        out = tree_attention(q, k, v, kc, vc, tables, lens, offsets, max_tokens=tokens, max_context=n,
                             scale=float(np.log(2.0)))
        w = (n - 1) * 2.0 ** -x
        want = w / (1 + w)
        tol = want * (U[dtype] + 2.0 ** -12) + (n * 2.0 ** -32 if dtype is torch.float16 else 0)
        tol += U[dtype] * (want + tol) + 2.0 ** -25
        assert ((out.double() - want).abs() <= tol).all(), (x, want, out.double().min().item(), out.double().max().item())


def test_padded_and_cut_batches(gpu):
    b = Batch(5, [40, 7, 0], [3, 70, 9], 16, 2, 128, 16, torch.float16, pad=6)
    out = torch.full(b.q.shape, 3.0, dtype=b.dtype, device=gpu)
    args = b.args(gpu)
    got = tree_attention(*args, out=out)
    assert got.data_ptr() == out.data_ptr()
    want = b.oracle()
    b.check(got, want)
    rest = torch.from_numpy(np.isnan(want[0])).to(gpu)  # rows 64.. of the second request, rows of none
    assert rest[:, 0, 0].nonzero().squeeze(1).tolist() == list(range(67, 73)) + list(range(82, 88)) and (out[rest] == 3).all()
    out.fill_(3)
    tree_attention(*args, out=out, max_tokens=4)
    want = b.oracle(max_tokens=4)
    b.check(out, want)
    assert (out[torch.from_numpy(np.isnan(want[0])).to(gpu)] == 3).all()
    # in place of q
    q = args[0].clone()
    tree_attention(q, *args[1:], out=q, max_context=0)
    b.check(q, b.oracle())


def test_absent_blocks_and_lengths_out_of_range(gpu):
    b = Batch(6, [100, 64, 50], [5, 33, 2], 16, 2, 128, 16, torch.bfloat16)
    b.tables[0, 2], b.tables[0, 6], b.tables[1, :], b.tables[2, 0] = -1, 2 ** 31 - 1, -5, b.kc.shape[0]
    b.check(tree_attention(*b.args(gpu)), b.oracle(), "absent blocks")
    b.lens = [10 ** 9, -4, 2 ** 31 - 1]  # cut to the table's columns; none
    want = b.oracle()
    b.check(tree_attention(*b.args(gpu)), want, "lengths")
    args = b.args(gpu)
    args[7] = torch.tensor([-3, 10 ** 6, 1, 7], dtype=torch.int32, device=gpu)
    assert tree_attention(*args).shape == b.q.shape
    args[8] = torch.full_like(args[8], 2 ** 31 - 1)
    args[7] = b.args(gpu)[7]
    b.parents = np.full(b.q.shape[0], -1)
    b.check(tree_attention(*args), b.oracle(), "parents out of range")


def test_what_is_not_seen_does_not_matter(gpu):
    """Infinities and NaN in the cache behind the length, in blocks of no table and in
    drafted tokens that a row does not descend from."""
    for dtype in (torch.bfloat16, torch.float16):
        b = Batch(7, [37, 0, 20], [6, 40, 34], 16, 2, 128, 16, dtype)
        used = {int(x) for x in b.tables.ravel() if x >= 0}
        for c in (b.kc, b.vc):
            for blk in set(range(c.shape[0])) - used:
                c[blk] = float("nan")
            c[int(b.tables[0, 2]), 5:] = float("inf")
            c[int(b.tables[2, 1]), 4:] = float("nan")
        b.check(tree_attention(*b.args(gpu)), b.oracle(), "behind the length")
        # tokens 0 (request 0), 7 and 39 (request 1) are not finite: only they and their descendants show it
        for row, value in ((0, float("nan")), (13, float("inf")), (45, -float("inf"))):
            b.v[row, :, 3:70] = value
        clean = Batch(7, [37, 0, 20], [6, 40, 34], 16, 2, 128, 16, dtype)
        for c, d in ((b.kc, clean.kc), (b.vc, clean.vc)):
            d.copy_(c)
        want = clean.oracle()
        got = tree_attention(*b.args(gpu)).cpu()
        for r in range(3):
            lo, hi = b.offsets[r], b.offsets[r + 1]
            see = D.ancestors(b.parents[lo:hi].tolist())
            for t in range(hi - lo):
                hit = [lo + j for j in see[t] if not torch.isfinite(b.v[lo + j]).all()]
                touched = torch.zeros(128, dtype=torch.bool)
                touched[3:70] = bool(hit)
                assert torch.equal(~torch.isfinite(got[lo + t]), touched.expand(16, 128)), (r, t)
                if len(hit) == 1:
                    assert torch.equal(torch.nan_to_num(got[lo + t, 0, 3:5].float(), nan=7.0),
                                       torch.nan_to_num(b.v[hit[0], 0, 3:5].float(), nan=7.0))
        got[~torch.isfinite(got)] = 0
        out = np.where(torch.isfinite(tree_attention(*b.args(gpu))).cpu().numpy(), want[0], 0)
        clean.check(got, (out, want[1], want[2]), "the rest")


@pytest.mark.parametrize("heads,tokens", [
    # few rows in one tile, in two of a wave, in two waves; two tiles of drafted tokens; through LDS
    ("0.5b", [2, 2, 1]), ("0.5b", [4, 4, 3]), ("0.5b", [9, 6, 7]), ("one", [6, 40, 34]), ("0.5b", [6, 40, 34]),
    ("3b", [2, 2, 1]), ("3b", [4, 3, 4]), ("3b", [8, 6, 7]), ("each", [6, 40, 34]), ("wide", [6, 40, 34])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_not_seen_does_not_matter_to_any_kernel(gpu, heads, tokens, dtype):
    h, kv, dim = HEADS[heads]
    lens, last = [37, 0, 20], dim - 9
    b, clean = (Batch(17, lens, tokens, h, kv, dim, 16, dtype) for _ in range(2))
    used = {int(x) for x in b.tables.ravel() if x >= 0}
    for c in (b.kc, b.vc):
        for blk in set(range(c.shape[0])) - used:
            c[blk] = float("nan")
        c[int(b.tables[0, 2]), 5:] = float("inf")
        c[int(b.tables[2, 1]), 4:] = float("nan")
    for row, value in ((0, float("nan")), (b.offsets[1] + 1, float("inf")), (b.offsets[2] - 1, -float("inf"))):
        b.v[row, :, 3:last] = value
    want = clean.oracle()
    got = tree_attention(*b.args(gpu), max_tokens=max(tokens)).cpu()
    for r in range(3):
        lo, hi = b.offsets[r], b.offsets[r + 1]
        see = D.ancestors(b.parents[lo:hi].tolist())
        for t in range(hi - lo):
            hit = [lo + j for j in see[t] if not torch.isfinite(b.v[lo + j]).all()]
            touched = torch.zeros(dim, dtype=torch.bool)
            touched[3:last] = bool(hit)
            assert torch.equal(~torch.isfinite(got[lo + t]), touched.expand(h, dim)), (r, t)
            if len(hit) == 1:
                assert torch.equal(torch.nan_to_num(got[lo + t, 0, 3:last].float(), nan=7.0),
                                   torch.nan_to_num(b.v[hit[0], 0, 3:last].float(), nan=7.0))
    rest = torch.isfinite(got)
    clean.check(torch.where(rest, got, 0), (np.where(rest.numpy(), want[0], 0), *want[1:]), "the rest")



def test_layouts_and_copies(gpu):
    b = Batch(8, [70, 20, 130], [3, 8, 1], 16, 2, 128, 16, torch.bfloat16)
    args = b.args(gpu)
    want = tree_attention(*args)
    b.check(want, b.oracle())
    # q, k and v as parts of one projection's rows
    n = b.q.shape[0]
    wide = torch.cat([t.reshape(n, -1) for t in args[:3]], 1)
    parts = [p.view(n, -1, 128) for p in wide.split([2048, 256, 256], 1)]
    assert torch.equal(tree_attention(*parts, *args[3:]), want)
    # one cache tensor, halves interleaved; heads in front of slots; wide table rows
    both = torch.stack(args[3:5], 1)
    assert torch.equal(tree_attention(*args[:3], both[:, 0], both[:, 1], *args[5:]), want)
    first = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in args[3:5]]
    assert torch.equal(tree_attention(*args[:3], *first, *args[5:]), want)
    table = torch.full((3, 50), -9, dtype=torch.int32, device=gpu)
    table[:, 7:7 + args[5].shape[1]] = args[5]
    assert torch.equal(tree_attention(*args[:5], table[:, 7:7 + args[5].shape[1]], *args[6:]), want)
    # a row stride of 1 element more, and a transposed head_dim: copied
    odd = torch.zeros(n, 2049, dtype=b.dtype, device=gpu)
    odd[:, 1:] = args[0].view(n, -1)
    turned = args[1].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(tree_attention(odd[:, 1:].view(n, 16, 128), turned, *args[2:]), want)
    # one row of keys for every token
    k1 = args[1][:1].expand(n, 2, 128)
    assert torch.equal(tree_attention(args[0], k1, *args[2:]), tree_attention(args[0], k1.contiguous(), *args[2:]))
    # nothing to do
    none = [a[:0] for a in args[:3]] + args[3:]
    none[7], none[8] = torch.zeros(4, dtype=torch.int32, device=gpu), None
    assert tree_attention(*none).shape == (0, 16, 128)


def test_cache_past_four_gigabytes(gpu):
    b = Batch(9, [100, 37], [4, 1], 8, 4, 128, 64, torch.bfloat16)
    args = b.args(gpu)
    big = [torch.empty(70000, 64, 4, 128, dtype=b.dtype, device=gpu) for _ in range(2)]  # 4.6 GB each
    shift = 70000 - b.kc.shape[0]
    for c, a in zip(big, args[3:5]):
        c[shift:] = a
    got = tree_attention(*args[:3], *big, torch.where(args[5] >= 0, args[5] + shift, -1), *args[6:])
    assert torch.equal(got, tree_attention(*args))


@pytest.mark.parametrize("heads,tokens", [("each", [1, 1]), ("3b", [4, 1]), ("0.5b", [9, 2]), ("3b", [40, 3])])
def test_cache_past_four_gigabytes_in_every_kernel(gpu, heads, tokens):
    h, kv, dim = HEADS[heads]
    b = Batch(19, [100, 37], tokens, h, kv, dim, 64, torch.bfloat16)
    args = b.args(gpu)
    blocks = (5 << 30) // (64 * kv * dim * 2)
    big = [torch.empty(blocks, 64, kv, dim, dtype=b.dtype, device=gpu) for _ in range(2)]  # 5 GiB each
    shift = blocks - b.kc.shape[0]
    for c, a in zip(big, args[3:5]):
        c[shift:] = a
    got = tree_attention(*args[:3], *big, torch.where(args[5] >= 0, args[5] + shift, -1), *args[6:], max_tokens=max(tokens))
    assert torch.equal(got, tree_attention(*args, max_tokens=max(tokens)))
    b.check(got, b.oracle())



def test_captured_and_replayed_with_other_lengths(gpu):
    """One graph serves steps whose lengths, trees and tables differ; two graphs on one
    pool and eager calls between do not disturb it."""
    steps = [Batch(20 + i, lens, tokens, 16, 2, 128, 16, torch.bfloat16, pad=24 - sum(tokens), columns=128)
             for i, (lens, tokens) in enumerate([([2000, 100, 5], [8, 8, 8]), ([3, 0, 2048], [1, 0, 12]),
                                                 ([500, 501, 502], [12, 1, 11])])]
    big = max(s.kc.shape[0] for s in steps)
    live = [torch.zeros_like(t) for t in steps[0].args(gpu)]
    live[3], live[4] = (torch.zeros(big, 16, 2, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def load(s):
        for dst, src in zip(live, s.args(gpu)):
            (dst[:src.shape[0]] if dst.dim() == 4 else dst).copy_(src)

    load(steps[0])
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(tree_attention(*live, max_tokens=12, max_context=2048))
        graphs.append(g)
    for turn in range(2):
        for s in steps:
            load(s)
            rows = s.offsets[-1]
            eager = tree_attention(*live, max_tokens=12, max_context=2048)[:rows].clone()
            s.check(torch.cat([eager, eager.new_zeros(24 - rows, 16, 128)]), s.oracle())
            for g, o in zip(graphs, outs):
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(o[:rows], eager)


@pytest.mark.parametrize("heads,tokens,context", [
    # rows of many parts (9000 keys), joined by sixteen waves; 12 rows and 3, 24, 64 and 128
    ("one", [1], None), ("3b", [1], None), ("each", [3], None), ("3b", [3], None), ("3b", [8], None), ("3b", [16], None),
    # the same call sized for a longer context: 33 to 64 rows through LDS, parts that stay empty
    ("3b", [5], 1 << 20), ("0.5b", [9], 1 << 20), ("3b", [2], 1 << 20), ("one", [64], 1 << 20), ("0.5b", [5], 1 << 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_parts(gpu, heads, tokens, context, dtype):
    b = Batch(30, [9000], tokens, *HEADS[heads], 16, dtype)
    b.check(tree_attention(*b.args(gpu), max_tokens=tokens[0], max_context=context), b.oracle())
    b = Batch(31, [40, 9000, 0, 700], [tokens[0], 1, tokens[0], 0], *HEADS[heads], 32, dtype)
    b.check(tree_attention(*b.args(gpu), max_tokens=tokens[0], max_context=context), b.oracle())


@pytest.mark.parametrize("requests,tokens,heads", [(1, 1, "0.5b"), (40, 4, "0.5b"), (300, 1, "one"), (2, 9, "0.5b"),
                                                   (3, 16, "3b"), (150, 40, "one"), (40, 17, "3b")])
def test_many_small_requests(gpu, requests, tokens, heads):
    """Grids on both sides of one workgroup per CU; units of less than a share and of several."""
    rng = np.random.default_rng(requests)
    b = Batch(32, rng.integers(0, 300, requests).tolist(), rng.integers(0, tokens + 1, requests).tolist(),
              *HEADS[heads], 16, torch.bfloat16)
    b.check(tree_attention(*b.args(gpu), max_tokens=tokens), b.oracle())


@pytest.mark.parametrize("requests,every,heads,long", [(600, 5, "one", (550,)), (1100, 9, "odd", (0, 700, 1060)),
                                                      (1100, 30, "wide", (511, 1024))])
def test_many_requests_through_lds(gpu, requests, every, heads, long):
    """More requests than the prefix sums take at a time (512), most of them without tokens, some
    of 40 and long ones on both sides of the bounds: their units are cut into shares and joined."""
    rng = np.random.default_rng(requests + every)
    tokens = np.where(np.arange(requests) % every == 3, rng.integers(0, 41, requests), 0)
    lens = rng.integers(0, 120, requests)
    lens[rng.random(requests) < 0.1] = 0
    for r in long:
        tokens[r], lens[r] = 37, 5000
    b = Batch(60, lens.tolist(), tokens.tolist(), *HEADS[heads], 16, torch.bfloat16)
    want = b.oracle()
    args = b.args(gpu)
    got = tree_attention(*args, max_tokens=40, max_context=5000)
    b.check(got, want)
    for _ in range(2):
        assert torch.equal(tree_attention(*args, max_tokens=40, max_context=5000), got)



@pytest.mark.parametrize("lens,tokens", [([300], [7]), ([5000, 20], [64, 5])])
def test_in_place(gpu, lens, tokens):
    b = Batch(33, lens, tokens, 16, 2, 128, 16, torch.bfloat16)
    args = b.args(gpu)
    want = tree_attention(*args)
    assert tree_attention(*args, out=args[0]) is not None and torch.equal(args[0], want)


@pytest.mark.parametrize("lens,tokens", [([40], [1]), ([900, 30], [1, 1]), ([60], [7])])
def test_default_bound_is_planned_as_the_rows(gpu, lens, tokens):
    """Without max_tokens: the same kernel, so the same bits, and no workspace for 64 tokens
    a request (68 MB) beside the output and what the few rows need."""
    b = Batch(34, lens, tokens, 16, 2, 128, 16, torch.bfloat16)
    args, rows = b.args(gpu), sum(tokens)
    want = tree_attention(*args, max_tokens=rows)
    b.check(want, b.oracle())
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = tree_attention(*args)
    assert torch.cuda.max_memory_allocated() - before < 4 << 20
    assert torch.equal(got, want)


def test_side_stream(gpu):
    b = Batch(11, [3000], [4], 16, 2, 128, 16, torch.bfloat16)
    args = b.args(gpu)
    want = tree_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [tree_attention(*args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("tokens", [1, 20])
def test_two_streams_at_once(gpu, tokens):
    """Split calls on two streams with nothing between them: each its own workspace."""
    args = [Batch(40 + s, [5000, 700], [tokens, 1], 16, 2, 128, 16, torch.bfloat16).args(gpu) for s in range(2)]
    want = [tree_attention(*a, max_tokens=tokens)[:tokens + 1] for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tree_attention(*args[i], max_tokens=tokens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_refusals(gpu):
    b = Batch(12, [20, 3], [2, 2], 16, 2, 128, 16, torch.bfloat16)
    good = b.args(gpu)

    def bad(error, match, at=None, value=None, **kw):
        args = list(good)
        if at is not None:
            args[at] = value
        with pytest.raises(error, match=match):
            tree_attention(*args, **kw)

    q, k, v, kc, vc, tables, lens, offsets, parents = good
    bad(RuntimeError, "ROCm GPU", 3, kc.cpu())
    bad(ValueError, "q on cpu", 0, q.cpu())
    bad(TypeError, "cache's dtype", 0, q.half())
    bad(ValueError, "q must be", 0, q[0])
    bad(ValueError, "k must be", 1, k[:3])
    bad(ValueError, "multiple of kv_heads", 0, q[:, :15])
    bad(ValueError, "agree", 4, vc[:1])
    bad(TypeError, "int32", 6, lens.long())
    bad(ValueError, "offsets", 7, offsets[:2])
    bad(ValueError, "parents", 8, parents[:2])
    bad(ValueError, "block_tables", 5, tables[:1])
    bad(ValueError, "max_tokens", max_tokens=0)
    bad(ValueError, "max_tokens", max_tokens=65)
    bad(ValueError, "scale", scale=float("nan"))
    bad(ValueError, "out must be", out=torch.empty_like(q)[:2])
    bad(ValueError, "out must be", out=torch.empty_like(q).float())
    bad(ValueError, "share memory", at=2, value=q[:, :2], out=q)
    small = [t[..., :32] for t in good[:5]] + good[5:]
    with pytest.raises(ValueError, match="head_dim"):
        tree_attention(*small)
    with pytest.raises(ValueError, match="multiple of 16"):
        tree_attention(*good[:3], kc[:, :8].contiguous(), vc[:, :8].contiguous(), *good[5:])
    shifted = torch.empty(kc.numel() + 1, dtype=kc.dtype, device=gpu)[1:].view(kc.shape)
    with pytest.raises(ValueError, match="aligned"):
        tree_attention(*good[:3], shifted, vc, *good[5:])
    with pytest.raises(ValueError, match="contiguous head_dim"):
        tree_attention(*good[:3], kc.transpose(1, 3), vc.transpose(1, 3), *good[5:])
    room = torch.zeros(5, 16, 128, dtype=torch.bfloat16, device=gpu)
    bad(ValueError, "a part of it", 0, room[:4], out=room[1:])
