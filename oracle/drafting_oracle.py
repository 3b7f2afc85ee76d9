"""CPU oracle of the paged cache and the 4-bit weights: plain loops and 64-bit
floats, from the operators' definitions (test infrastructure only)."""

from __future__ import annotations

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
#: signed values of the codes 0..15
CODES = np.concatenate([VALUES, -VALUES])


def bf16(a) -> np.ndarray:
    """float32 values rounded to bf16 (nearest, ties to even), NaN kept."""
    a = np.asarray(a, dtype=np.float32)
    bits = a.view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(a), a, out)


def quantize4(w: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [n, k], scale float32 [n, groups]) of a float32 weight."""
    w = np.asarray(w, dtype=np.float32)
    n, k = w.shape
    groups = -(-k // group)
    codes, scale = np.zeros((n, k), np.uint8), np.zeros((n, groups), np.float32)
    for g in range(groups):
        part = w[:, g * group:(g + 1) * group].astype(np.float64)
        a = np.abs(part)
        with np.errstate(invalid="ignore"):
            top = a.max(axis=1)  # NaN stays
            s = bf16(np.where(np.isnan(top), np.float32(np.nan), np.maximum(top, np.float64(np.float32(1e-8))))
                     .astype(np.float32) / np.float32(6.0))
        scale[:, g] = s
        s = s.astype(np.float64)[:, None]
        c = np.zeros(part.shape, np.uint8)
        for i in range(7):
            # between the values i and i + 1: an even i keeps its midpoint
            mid = (VALUES[i] + VALUES[i + 1]) / 2
            with np.errstate(invalid="ignore"):
                c += (a > mid * s) if i % 2 == 0 else (a >= mid * s)
        codes[:, g * group:(g + 1) * group] = c + 8 * ((part < 0) & (c > 0))
    return codes, scale


def dense4(codes: np.ndarray, scale: np.ndarray, group: int) -> np.ndarray:
    """value * scale, exact in float64."""
    per = np.repeat(scale.astype(np.float64), group, axis=1)[:, :codes.shape[1]]
    with np.errstate(invalid="ignore"):
        return CODES[codes] * per


def append(lens, new, offsets, tables, free, count, bs, rows, index=None):
    """append_blocks on Python lists, in place -> (slots, status, free count)."""
    status, before = [], list(lens)
    asked = 0
    for b in range(len(lens)):
        add = max(new[b], 0)
        have, want = -(-lens[b] // bs), -(-(lens[b] + add) // bs)
        if lens[b] < 0 or want > len(tables[b]):
            status.append(2)
            continue
        asked += want - have
        if want > have and asked > count:
            status.append(1)
            continue
        status.append(0)
        for j in range(have, want):
            tables[b][j] = free[count - 1 - (asked - (want - have)) - (j - have)]
        lens[b] += add
    used = sum(-(-lens[b] // bs) - -(-before[b] // bs) for b in range(len(lens)) if status[b] == 0)
    slots = [-1] * rows
    for b in range(len(lens)):
        if status[b]:
            continue
        for i in range(offsets[b], min(offsets[b + 1], rows)):
            n = index[i] if index is not None else i - offsets[b]
            if 0 <= n < max(new[b], 0):
                pos = before[b] + n
                block = tables[b][pos // bs]
                if block >= 0:
                    slots[i] = block * bs + pos % bs
    return slots, status, count - used


def truncate(lens, keep, tables, free, count, bs):
    """truncate_blocks on Python lists, in place -> free count."""
    back = []
    for b in range(len(lens)):
        have = min(-(-max(lens[b], 0) // bs), len(tables[b]))
        lens[b] = min(max(keep[b], 0), max(lens[b], 0))
        left = min(-(-lens[b] // bs), have)
        back += [block for block in tables[b][left:have] if block >= 0]
        tables[b][left:have] = [-1] * (have - left)
    for e, block in enumerate(back):
        at = count + len(back) - 1 - e
        if at < len(free):
            free[at] = block
    return min(count + len(back), len(free))


def ancestors(parents) -> list[set]:
    """For each token of a request the tokens it sees: itself and its ancestors."""
    out = []
    for t in range(len(parents)):
        see, j = set(), t
        while True:
            see.add(j)
            if not 0 <= parents[j] < j:
                break
            j = parents[j]
        out.append(see)
    return out


def tree_attention(q, k, v, kc, vc, tables, lens, offsets, parents, scale, max_tokens=64):
    """float64 (out, spread, reach) of the batch, NaN where a row belongs to no
    request.  spread: sum of weight * (|v| + |out|), what a relative error of the
    weights is multiplied by; reach [rows, heads]: the largest scale * sum |q||k|
    over the keys seen."""
    rows, heads, dim = q.shape
    per = heads // k.shape[1]
    bs, blocks = kc.shape[1], kc.shape[0]
    out = np.full(q.shape, np.nan)
    spread, reach = np.zeros(q.shape), np.zeros((rows, heads))
    for b in range(len(lens)):
        lo, hi = offsets[b], min(offsets[b + 1], rows)
        tokens = min(hi - lo, max_tokens)
        places = [(int(tables[b][p // bs]), p % bs) for p in range(min(max(lens[b], 0), len(tables[b]) * bs))]
        places = [p for p in places if 0 <= p[0] < blocks]
        blk, at = (np.array([p[i] for p in places], dtype=np.int64) for i in (0, 1))
        see = ancestors([(parents[lo + t] if parents is not None else t - 1) for t in range(tokens)])
        for t in range(tokens):
            own = lo + np.array(sorted(see[t]))
            for h in range(heads):
                kv = h // per
                key = np.concatenate([kc[blk, at, kv], k[own, kv]])
                val = np.concatenate([vc[blk, at, kv], v[own, kv]])
                s = scale * (key @ q[lo + t, h])
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ val
                out[lo + t, h] = o
                spread[lo + t, h] = w @ np.abs(val) + np.abs(o)
                reach[lo + t, h] = abs(scale) * (np.abs(key) @ np.abs(q[lo + t, h])).max()
    return out, spread, reach
