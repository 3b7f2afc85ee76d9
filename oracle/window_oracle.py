"""CPU oracle of the operators of long texts in a bounded cache: 64-bit floats, from
the operators' definitions (test infrastructure only)."""

from __future__ import annotations

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def cut6(x) -> np.ndarray:
    """The first 6 significant bits of float32 numbers at least 0; NaN and infinity stay."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(invalid="ignore"):
        m, e = np.frexp(x)
        return np.where(np.isfinite(x), np.ldexp(np.floor(m * 64) / 64, e), x).astype(np.float32)


def quantize_rows(x) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8, scale float32 [..., dim / 32]) of float32 rows [..., dim]."""
    x = np.asarray(x, dtype=np.float32)
    f = x.reshape(*x.shape[:-1], -1, 32).astype(np.float64)
    a = np.abs(f)
    with np.errstate(invalid="ignore"):
        top = a.max(-1)  # NaN stays
        floor = np.float64(np.float32(1e-8))
        s32 = cut6(np.where(np.isnan(top), np.nan, np.maximum(top, floor)).astype(np.float32) / np.float32(6.0))
        s = s32.astype(np.float64)[..., None]
        c = np.zeros(f.shape, np.uint8)
        for i in range(7):
            # between the values i and i + 1: an even i keeps its midpoint
            mid = (VALUES[i] + VALUES[i + 1]) / 2
            c += (a > mid * s) if i % 2 == 0 else (a >= mid * s)
    return (c + 8 * ((f < 0) & (c > 0))).reshape(x.shape).astype(np.uint8), s32


def dense_rows(codes, scale) -> np.ndarray:
    """value * scale, exact in float64."""
    value = np.concatenate([VALUES, -VALUES])
    with np.errstate(invalid="ignore"):
        return value[codes] * np.repeat(np.asarray(scale, np.float64), 32, axis=-1)


def sees(n, length, window=None, sinks=0) -> np.ndarray:
    """[n, length]: which tokens the n newest rows of a text see."""
    p = np.arange(length - n, length)[:, None]
    j = np.arange(length)
    near = np.ones((n, length), bool) if window is None else (j > p - window) | (j < sinks)
    return (j <= p) & near


def places(table, length, bs, blocks):
    """(block or -1, place in it) of a request's tokens."""
    j = np.arange(length)
    blk = np.asarray(table)[j // bs].astype(np.int64) if length else j
    return np.where((blk >= 0) & (blk < blocks), blk, -1), j % bs


def attention(q, kc, vc, tables, lens, offsets, scale, window=None, sinks=0, max_tokens=None):
    """float64 (out, lse, spread, mass, reach) of a batch over dense caches, NaN where a row
    belongs to no request (zeros and -inf where it sees nothing).  mass: sum of weight * |v|;
    spread: that plus |out|, what a relative error of the weights is multiplied by; reach
    [rows, heads]: the largest scale * sum |q||k| over the tokens seen."""
    rows, heads, dim = q.shape
    per, bs, blocks = heads // kc.shape[2], kc.shape[1], kc.shape[0]
    out, lse = np.full(q.shape, np.nan), np.full((rows, heads), np.nan)
    spread, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads))
    for b in range(len(lens)):
        lo, hi = offsets[b], min(offsets[b + 1], rows)
        n = hi - lo
        length = min(max(lens[b], 0), len(tables[b]) * bs)
        blk, at = places(tables[b], length, bs, blocks)
        see = sees(n, length, window, sinks) & (blk >= 0)
        few = n if max_tokens is None else min(n, max_tokens)
        for h in range(heads):
            key, val = kc[blk, at, h // per], vc[blk, at, h // per]
            for t in range(few):
                m = see[t]
                out[lo + t, h], lse[lo + t, h] = 0, -np.inf
                if not m.any():
                    continue
                k, v = key[m], val[m]
                s = scale * (k @ q[lo + t, h])
                top = s.max()
                w = np.exp(s - top)
                lse[lo + t, h] = np.log(w.sum()) + top
                w /= w.sum()
                out[lo + t, h] = w @ v
                mass[lo + t, h] = w @ np.abs(v)
                spread[lo + t, h] = mass[lo + t, h] + np.abs(out[lo + t, h])
                reach[lo + t, h] = abs(scale) * (np.abs(k) @ np.abs(q[lo + t, h])).max()
    return out, lse, spread, mass, reach


def accumulate(weights, q, kc, tables, lens, offsets, lse, scale, new_lens=None, window=None, sinks=0):
    """accumulate_weights on a float64 copy -> (weights, reach): reach per slot, the largest
    scale * sum |q||k| + |lse| of what was added."""
    weights, rows = weights.astype(np.float64).copy(), q.shape[0]
    far = np.zeros_like(weights)
    heads = q.shape[1]
    per, bs, blocks = heads // kc.shape[2], kc.shape[1], kc.shape[0]
    for b in range(len(lens)):
        lo, hi = offsets[b], min(offsets[b + 1], rows)
        n, length = hi - lo, min(max(lens[b], 0), len(tables[b]) * bs)
        blk, at = places(tables[b], length, bs, blocks)
        see = sees(n, length, window, sinks)
        for j in range(length):
            if blk[j] < 0:
                continue
            if new_lens is not None and j >= length - max(new_lens[b], 0):
                weights[blk[j], at[j]] = 0
            t = np.nonzero(see[:, j])[0]
            for h in range(heads):
                k = kc[blk[j], at[j], h // per]
                weights[blk[j], at[j]] += np.exp(scale * (q[lo + t, h] @ k) - lse[lo + t, h]).sum()
                if len(t):
                    r = abs(scale) * (np.abs(q[lo + t, h]) @ np.abs(k)) + np.abs(lse[lo + t, h])
                    far[blk[j], at[j]] = max(far[blk[j], at[j]], r.max())
    return weights, far


def stays(weights, length, budget, sinks=0, recent=0) -> list[int]:
    """The tokens of a request that stay, in order; weights: one per token (an absent
    token's is None)."""
    most = max(budget, 0)
    if length <= most:
        return list(range(length))
    sinks = min(sinks, most)
    recent = min(recent, most - sinks)

    def rank(i):
        w = weights[i]
        return (2, 0.0, i) if w is None else (0, 0.0, i) if w != w else (1, -w, i)

    others = sorted(range(sinks, length - recent), key=rank)[:most - sinks - recent]
    return list(range(sinks)) + sorted(others) + list(range(length - recent, length))


def evict(weights, tables, lens, budget, caches, sinks=0, recent=0, max_context=None) -> list[int]:
    """evict_tokens in place on numpy arrays [blocks, block_size, ...] -> kept."""
    blocks, bs = weights.shape
    kept = []
    for b in range(len(lens)):
        length = min(max(lens[b], 0), len(tables[b]) * bs)
        if max_context is not None and length > max_context:
            kept.append(length)
            continue
        blk, at = places(tables[b], length, bs, blocks)
        w = [float(weights[x, y]) if x >= 0 else None for x, y in zip(blk, at)]
        stay = stays(w, length, budget[b], sinks, recent)
        kept.append(len(stay))
        for array in [weights, *caches]:
            old = array.copy()
            for i, j in enumerate(stay):
                if i != j and blk[i] >= 0 and blk[j] >= 0:
                    array[blk[i], at[i]] = old[blk[j], at[j]]
    return kept
