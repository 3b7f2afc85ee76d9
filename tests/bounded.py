"""Batches over the 16-bit and the 4-bit cache for the tests of the operators of long
texts, and the bounds that their results are held to.

A score is a sum of D exact products, each addition off by at most 2^-23 of the
magnitudes (in 4 bits of values * q: the scale is a factor of both), then scaled: off by
(D + 8) 2^-23 reach, reach = scale max sum |q||k|.  So a weight p = 2^(score - m) is off by
a factor of 1 + e, e = (D + 12) 2^-23 reach + 2^-20 (the rounding of c and of the
exponent lies in reach; v_exp_f32 and the rescaling by a few more units); its rounding to
the type t by u = half a step of t.  fp32 additions in each of keys / 32 steps and in the
joins: (keys / 32 + 64) 2^-23.

16 bits: out = sum p v / sum p, p rounded above, and below either the same or unrounded:
off by (u + e) sum w (|v| + |out|).  A p that fp16 rounds to a multiple of 2^-24 may be
off by 2^-25 instead, times at most `keys` against a sum of at least 1.  Many rows over the
4-bit cache are the same (its values are exact in both types).
4 bits, single rows: the numerator's p * scale is rounded to bf16 (for fp16 rows in two
terms, off by 2^-17), the sum is of the weights before that: u sum w |v| and e as above.
Both: then the output's own rounding.
lse: off by e, and the logarithm and the two roundings behind it by 4 units of 2^-24 of it."""

from __future__ import annotations

import numpy as np
import torch

from oracle import window_oracle as W
from pageserve_amd import KVCache4, write_kv4

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}

HEADS = {"3b": (16, 2, 128), "0.5b": (14, 2, 64), "one": (1, 1, 64), "each": (4, 4, 128), "wide": (24, 1, 128),
         "odd": (15, 3, 64)}


class Batch:
    """Requests of tokens[b] rows at the end of lens[b] cached tokens, on the CPU; whatever no
    request owns in the cache holds `garbage` (None: ordinary numbers)."""

    def __init__(self, seed, lens, tokens, heads, kv, dim, bs, dtype, bits=16, pad=0, columns=None, garbage=None):
        rng = np.random.default_rng(seed)
        self.heads, self.kv, self.dim, self.bs, self.dtype, self.bits = heads, kv, dim, bs, dtype, bits
        self.lens, self.offsets = list(lens), np.concatenate([[0], np.cumsum(tokens)]).astype(int).tolist()
        rows = self.offsets[-1] + pad

        def values(*shape):
            return torch.from_numpy(rng.standard_normal(shape)).to(dtype)

        self.q = values(rows, heads, dim)
        have = [-(-max(n, 0) // bs) for n in lens]
        self.blocks = sum(have) + 2
        self.kc, self.vc = values(self.blocks, bs, kv, dim), values(self.blocks, bs, kv, dim)
        order, at = rng.permutation(self.blocks).tolist(), 0
        columns = columns if columns is not None else max(have + [0])
        self.tables = np.full((len(have), columns), -1, dtype=np.int32)
        owned = np.zeros((self.blocks, bs), bool)
        for b, h in enumerate(have):
            self.tables[b, :h] = order[at:at + h]
            at += h
            j = np.arange(max(lens[b], 0))
            owned[self.tables[b, j // bs], j % bs] = True
        self.owned = torch.from_numpy(owned)
        if garbage is not None:
            self.kc[~self.owned] = garbage
            self.vc[~self.owned] = garbage

    def ints(self, gpu, a):
        return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(gpu)

    def dense(self):
        """The caches that the kernels see, float64 [blocks, block_size, kv_heads, head_dim]."""
        f = [x.to(torch.float32).numpy() for x in (self.kc, self.vc)]
        return [W.dense_rows(*W.quantize_rows(x)) if self.bits == 4 else x.astype(np.float64) for x in f]

    def cache(self, gpu):
        """On the GPU: (k_cache, v_cache), or the 4-bit cache of the same rows, written by write_kv4."""
        k, v = self.kc.to(gpu), self.vc.to(gpu)
        if self.bits == 16:
            return k, v
        c = KVCache4(self.blocks, self.bs, self.kv, self.dim, gpu)
        write_kv4(k.flatten(0, 1), v.flatten(0, 1), c, torch.arange(self.blocks * self.bs, device=gpu))
        return (c,)

    def args(self, gpu):
        return [self.q.to(gpu), *self.cache(gpu), self.ints(gpu, self.tables), self.ints(gpu, self.lens),
                self.ints(gpu, self.offsets)]

    def oracle(self, scale=None, window=None, sinks=0, max_tokens=None):
        return W.attention(self.q.to(torch.float64).numpy(), *self.dense(), self.tables, self.lens, self.offsets,
                           self.dim ** -0.5 if scale is None else scale, window, sinks, max_tokens)

    def factor(self, reach):
        """e of every row and head"""
        keys = max(self.lens + [0])
        return (self.dim + 12) * 2.0 ** -23 * reach + 2.0 ** -20 + (keys / 32 + 64) * 2.0 ** -23

    def check(self, got, want, what=""):
        """got: the output, or (output, lse)"""
        out, lse, spread, _, reach = want
        got, got_lse = got if isinstance(got, tuple) else (got, None)
        assert got.dtype == self.dtype
        got = got.to(torch.float64).cpu().numpy()
        live = ~np.isnan(lse)
        u, e = U[self.dtype], self.factor(reach)
        if got_lse is not None:
            g = got_lse.to(torch.float64).cpu().numpy()
            none = live & np.isneginf(lse)
            assert np.isneginf(g[none]).all(), f"{what}: lse of rows that see nothing"
            some = live & ~none
            off = np.abs(g[some] - lse[some]) - (e[some] + 2.0 ** -22 * np.abs(lse[some]))
            assert (off <= 0).all(), f"{what}: lse {off.max():.3g} over the bound"
        e = e[..., None] + (max(self.lens + [0]) * 2.0 ** -25 if self.dtype is torch.float16 else 0)
        tol = (u + e) * spread
        tol = tol + u * (np.abs(out) + tol) + 2.0 ** -25
        off = np.where(live[..., None], np.abs(got - out) - tol, -1)
        assert not np.isnan(off).any(), f"{what}: not a number"
        assert (off <= 0).all(), f"{what}: {off.max():.3g} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
