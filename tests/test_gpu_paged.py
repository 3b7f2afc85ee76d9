"""Block tables, slots and cache rows on the GPU against the oracle's loops: whole
numbers, so every comparison is for equality."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafting_oracle as D
from pageserve_amd import append_blocks, truncate_blocks, write_kv

pytestmark = pytest.mark.gpu


def _i32(a, gpu):
    return torch.tensor(a, dtype=torch.int32, device=gpu)


class _State:
    """The same bookkeeping twice: Python lists, and tensors on the GPU."""

    def __init__(self, gpu, lens, columns, bs, spare, seed=0, stride=None):
        rng = np.random.default_rng(seed)
        have = [-(-max(n, 0) // bs) for n in lens]
        pool = rng.permutation(sum(have) + spare).tolist()
        self.gpu, self.bs = gpu, bs
        self.tables, at = [], 0
        for h in have:
            self.tables.append((pool[at:at + h] + [-1] * columns)[:columns])
            at += h
        self.lens, self.count = list(lens), spare
        self.free = pool[at:] + [-7] * (len(pool) - spare)
        wide = torch.full((len(lens), stride or columns), -3, dtype=torch.int32, device=gpu)
        wide[:, :columns] = _i32(self.tables, gpu).view(len(lens), columns)
        self.wide, self.t = wide, wide[:, :columns]
        self.l, self.f, self.c = _i32(self.lens, gpu), _i32(self.free, gpu), _i32([self.count], gpu)

    def append(self, new, offsets, rows, index=None):
        want = D.append(self.lens, new, offsets, self.tables, self.free, self.count, self.bs, rows, index)
        self.count = want[2]
        slots, status = append_blocks(self.l, _i32(new, self.gpu), _i32(offsets, self.gpu), self.t, self.f, self.c,
                                      self.bs, rows, index=None if index is None else _i32(index, self.gpu))
        assert slots.dtype == torch.int64 and status.dtype == torch.int32
        assert status.tolist() == want[1]
        assert slots.tolist() == want[0]
        self.same()
        return want

    def truncate(self, keep):
        self.count = D.truncate(self.lens, keep, self.tables, self.free, self.count, self.bs)
        truncate_blocks(self.l, _i32(keep, self.gpu), self.t, self.f, self.c, self.bs)
        self.same()

    def same(self):
        assert self.l.tolist() == self.lens and self.c.item() == self.count
        assert self.t.tolist() == self.tables and self.f.tolist() == self.free


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).tolist()


@pytest.mark.parametrize("requests,tokens,bs", [(1, 1, 16), (1, 5000, 16), (3, 7, 1), (8, 12, 16), (100, 3, 5), (70, 100, 64),
                                                (1500, 2, 16), (4096, 1, 128)])
@pytest.mark.parametrize("indexed", [False, True])
def test_append_then_truncate(gpu, requests, tokens, bs, indexed):
    rng = np.random.default_rng(requests + tokens)
    lens = rng.integers(0, 60, requests).tolist()
    counts = rng.integers(0, tokens + 1, requests).tolist()
    offsets = _offsets(counts)
    rows = offsets[-1] + 5  # a padded batch
    new, index = counts, None
    if indexed:
        index = [-1] * rows
        new = []
        for b, c in enumerate(counts):
            kept = np.flatnonzero(rng.random(c) < 0.4)
            for n, i in enumerate(kept):
                index[offsets[b] + i] = n
            new.append(len(kept))
        index[-1] = 0
    columns = -(-(60 + tokens) // bs)
    s = _State(gpu, lens, columns, bs, spare=requests * (tokens // bs + 2), stride=columns + 3)
    before = (list(s.lens), [list(t) for t in s.tables], list(s.free), s.count)
    got = s.append(new, offsets, rows, index)
    assert not any(got[1]) and (s.wide[:, columns:] == -3).all()
    used = [x for x in got[0] if x >= 0]
    assert len(set(used)) == len(used) == (sum(new))
    s.truncate(before[0])
    assert before == (s.lens, s.tables, s.free, s.count)
    s.append(new, offsets, rows, index)
    s.truncate([0] * requests)
    assert s.count == len(s.free) and sorted(s.free) == list(range(len(s.free)))


@pytest.mark.parametrize("requests,columns", [(1, 5), (3, 3), (40, 30), (700, 7)])
def test_holes_are_not_given_back(gpu, requests, columns):
    """Absent blocks below the length: the stack gets the others, in order, and nothing
    that append hands out afterwards is absent."""
    rng = np.random.default_rng(columns)
    lens = rng.integers(0, 4 * columns + 1, requests).tolist()
    lens[0] = 4 * columns
    s = _State(gpu, lens, columns, 4, spare=3, seed=requests)
    holes = 0
    for b, n in enumerate(lens):
        for c in range(-(-n // 4)):
            if rng.random() < 0.4 or (b, c) == (0, 1):
                s.tables[b][c], holes = -1 - c, holes + 1
    s.t.copy_(_i32(s.tables, gpu))
    s.truncate([n // 2 for n in lens])
    s.truncate([0] * requests)
    assert s.count == len(s.free) - holes and min(s.free[:s.count]) >= 0
    new = [min(4 * columns, 4 * s.count)] + [0] * (requests - 1)
    slots, status, _ = s.append(new, _offsets(new), new[0])
    assert status == [0] * requests and min(slots) >= 0 and len(set(slots)) == new[0]
    # a stack that is too short keeps what was on it and drops the last that come
    s = _State(gpu, [8, 9], 3, 4, spare=0)
    s.free, s.f = s.free[:2], s.f[:2].contiguous()
    s.tables[0][0] = -1
    s.t.copy_(_i32(s.tables, gpu))
    s.truncate([0, 0])


def test_too_few_blocks_columns_and_odd_lengths(gpu):
    for spare in range(0, 9):
        s = _State(gpu, [4, 15, 16, 0, 31, 40], 4, 16, spare=spare, seed=spare)
        s.append([13, 1, 20, 0, 40, 30], _offsets([13, 1, 20, 0, 40, 30]), 104)
    s = _State(gpu, [5, 10, 3, 8], 3, 4, spare=20)
    s.lens[1] = -2
    s.l[1] = -2
    s.append([-4, 3, 2, 1], _offsets([2, 3, 2, 1]), 8)
    s.truncate([-1, 5, 100, 3])
    # no table columns, no free list
    s = _State(gpu, [0, 0], 0, 16, spare=0)
    s.append([1, 0], [0, 1, 1], 1)
    s.truncate([0, 0])


def test_lengths_at_the_largest(gpu):
    lens, new = _i32([2 ** 31 - 3, 5], gpu), _i32([10, 2 ** 31 - 1], gpu)
    tables, free, count = _i32([[1] * 3] * 2, gpu), _i32([0, 4], gpu), _i32([2], gpu)
    slots, status = append_blocks(lens, new, _i32([0, 1, 2], gpu), tables, free, count, 65536, 2)
    assert status.tolist() == [2, 2] and slots.tolist() == [-1, -1]
    assert lens.tolist() == [2 ** 31 - 3, 5] and count.item() == 2
    count.fill_(99)  # above the list's capacity: cut to it
    slots, status = append_blocks(lens, _i32([0, 65536 * 2 - 5], gpu), _i32([0, 0, 2], gpu), tables, free, count, 65536, 2)
    assert status.tolist() == [2, 0] and count.item() == 1 and tables[1].tolist() == [1, 4, 1]


def test_wrong_offsets_stay_inside(gpu):
    lens, new = _i32([3, 3], gpu), _i32([4, 4], gpu)
    tables, free, count = _i32([[0, -1], [1, -1]], gpu), _i32([2, 3], gpu), _i32([2], gpu)
    slots, _ = append_blocks(lens, new, _i32([900, -5, 2 ** 31 - 1], gpu), tables, free, count, 4, 6)
    assert slots.numel() == 6 and ((slots >= -1) & (slots < 16)).all()


def test_arrays_that_share_memory_are_refused(gpu):
    """What a call writes shares no element with its other arrays; parts of one buffer,
    between a table's rows too, are fine."""
    buf = torch.zeros(200, dtype=torch.int32, device=gpu)
    table = buf[100:148].view(4, 12)[:, :5]  # rows of 5, 12 apart
    good = dict(lens=buf[:4], new_lens=buf[4:8], offsets=buf[8:13], block_tables=table, free_blocks=buf[20:40],
                free_count=buf[40:41], block_size=16, rows=3, index=buf[41:44])
    append_blocks(**good)
    append_blocks(**{**good, "lens": buf[105:109], "new_lens": buf[117:121], "free_blocks": buf[129:136]})
    for kw in (dict(new_lens=buf[:4]), dict(new_lens=buf[3:7]), dict(offsets=buf[2:7]), dict(index=buf[3:6]),
               dict(free_blocks=buf[:4]), dict(free_count=buf[1:2]), dict(lens=buf[100:104]), dict(lens=buf[97:101]),
               dict(lens=buf[109:113]), dict(new_lens=buf[116:120]), dict(offsets=buf[136:141]),
               dict(offsets=buf[140:145]), dict(free_blocks=buf[90:190]), dict(free_blocks=buf[105:125]),
               dict(index=buf[40:43])):
        with pytest.raises(ValueError, match="share memory"):
            append_blocks(**{**good, **kw})
    keep = dict(lens=buf[:4], keep=buf[4:8], block_tables=table, free_blocks=buf[20:40], free_count=buf[40:41], block_size=16)
    truncate_blocks(**keep)
    truncate_blocks(**{**keep, "keep": buf[:4]})
    for kw in (dict(keep=buf[1:5]), dict(keep=buf[101:105]), dict(free_blocks=buf[:20]), dict(free_blocks=buf[40:50]),
               dict(free_count=buf[112:113]), dict(lens=buf[20:24]), dict(keep=buf[38:42])):
        with pytest.raises(ValueError, match="share memory"):
            truncate_blocks(**{**keep, **kw})
    # tables of one row and of one column
    one = dict(good, lens=buf[:1], new_lens=buf[1:2], offsets=buf[2:4], block_tables=buf[4:9].view(1, 5))
    append_blocks(**one)
    with pytest.raises(ValueError, match="share memory"):
        append_blocks(**{**one, "index": buf[8:11]})


def test_append_replayed_with_other_lengths(gpu):
    s = _State(gpu, [3, 20, 0], 8, 4, spare=18)
    new, offsets = _i32([0, 0, 0], gpu), _i32([0, 0, 0, 0], gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        slots, status = append_blocks(s.l, new, offsets, s.t, s.f, s.c, 4, 9)
    for counts in ([2, 3, 4], [0, 1, 0], [5, 0, 3], [1, 1, 1]):
        new.copy_(_i32(counts, gpu))
        offsets.copy_(_i32(_offsets(counts), gpu))
        g.replay()
        want = D.append(s.lens, counts, _offsets(counts), s.tables, s.free, s.count, 4, 9)
        s.count = want[2]
        assert slots.tolist() == want[0] and status.tolist() == want[1]
        s.same()


def _reference_write(k, v, kc, vc, slots):
    bs = kc.shape[1]
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < kc.shape[0] * bs:
            kc[s // bs, s % bs] = k[i]
            vc[s // bs, s % bs] = v[i]


@pytest.mark.parametrize("rows,heads,dim,bs", [(1, 2, 128, 16), (7, 2, 64, 16), (300, 8, 128, 64), (33, 1, 96, 1), (5, 3, 20, 7),
                                               (2000, 2, 128, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_kv(gpu, rows, heads, dim, bs, dtype):
    gen = torch.Generator().manual_seed(rows + dim)
    blocks = rows // bs + 3
    k, v = (torch.randn(rows, heads, dim, generator=gen).to(dtype) for _ in range(2))
    slots = torch.randperm(blocks * bs, generator=gen)[:rows]
    slots[torch.rand(rows, generator=gen) < 0.3] = -1
    if rows > 4:
        slots[0], slots[1], slots[2] = blocks * bs, 2 ** 40, -(2 ** 40)
    base = torch.randn(2, blocks, bs, heads, dim, generator=gen).to(dtype)
    want = base.clone()
    _reference_write(k, v, want[0], want[1], slots)
    layouts = {
        "two halves": lambda: base.to(gpu),
        "interleaved": lambda: base.to(gpu).transpose(0, 1).contiguous().transpose(0, 1),
        "heads first": lambda: base.to(gpu).transpose(2, 3).contiguous().transpose(2, 3),
        "one element off": lambda: torch.empty(base.numel() + 1, dtype=dtype, device=gpu)[1:].view(base.shape).copy_(
            base),
    }
    for name, make in layouts.items():
        c = make()
        assert write_kv(k.to(gpu), v.to(gpu), c[0], c[1], slots.to(gpu)) is None
        assert torch.equal(c.cpu(), want), name
    # rows that are parts of a wider projection, and rows whose last dimension is not contiguous
    wide = torch.zeros(rows, 3 * heads * dim, dtype=dtype, device=gpu)
    wide[:, heads * dim:2 * heads * dim] = k.view(rows, -1).to(gpu)
    turned = v.to(gpu).transpose(1, 2).contiguous().transpose(1, 2)
    c = base.to(gpu)
    write_kv(wide[:, heads * dim:2 * heads * dim].view(rows, heads, dim), turned, c[0], c[1], slots.to(gpu))
    assert torch.equal(c.cpu(), want)


@pytest.mark.parametrize("dim", [64, 20])  # 16-byte pieces, single elements
def test_rows_moved_within_the_cache(gpu, dim):
    base = torch.randn(2, 300, 16, 2, dim, generator=torch.Generator().manual_seed(dim)).bfloat16()
    slots = torch.randperm(4800, generator=torch.Generator().manual_seed(1))
    slots[::7] = -1
    shift = torch.arange(1, 4801)  # every row to its neighbour's place, the last one out
    for s in (slots, shift):
        c = base.to(gpu)
        rows = c.flatten(1, 2)
        write_kv(rows[0], rows[1], c[0], c[1], s.to(gpu))
        want = base.clone()
        _reference_write(base[0].flatten(0, 1), base[1].flatten(0, 1), want[0], want[1], s)
        assert torch.equal(c.cpu(), want)
    # keys from the value cache and values from the key cache
    c = base.to(gpu)
    rows = c.flatten(1, 2)
    write_kv(rows[1, :40], rows[0, 8:48], c[0], c[1], shift[:40].to(gpu))
    want = base.clone()
    _reference_write(base[1].flatten(0, 1)[:40], base[0].flatten(0, 1)[8:48], want[0], want[1], shift[:40])
    assert torch.equal(c.cpu(), want)


def test_caches_that_overlap_themselves_are_refused(gpu):
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=gpu)
    k, s = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=gpu), torch.arange(3, device=gpu)
    for bad in (c[:1].expand(4, 16, 2, 64), c[:, :1].expand(4, 16, 2, 64), c[:, :, :1].expand(4, 16, 2, 64),
                c.view(-1).as_strided((4, 16, 2, 64), (1024, 128, 64, 1))):
        for pair in ((bad, c), (c, bad)):
            with pytest.raises(ValueError, match="overlap itself"):
                write_kv(k, k, *pair, s)
    assert not c.any()
    # one block, one slot, one head: a step of any size
    one = c[:1, :1, :1].expand(1, 1, 1, 64)
    write_kv(k[:1, :1], k[:1, :1], one, one, s[:1])
    assert c.sum() == 64


def test_write_past_four_gigabytes(gpu):
    c = torch.empty(40000, 64, 8, 128, dtype=torch.bfloat16, device=gpu)  # 5.2 GB
    k = torch.randn(3, 8, 128, device=gpu).bfloat16()
    slots = torch.tensor([40000 * 64 - 1, 39999 * 64, 5], device=gpu)
    write_kv(k, k, c, c, slots)
    assert torch.equal(c.view(-1, 8, 128)[slots], k)


def test_refusals(gpu):
    i = lambda *a: _i32(list(a), gpu)  # noqa: E731
    good = dict(lens=i(1), new_lens=i(1), offsets=i(0, 1), block_tables=_i32([[0, -1]], gpu), free_blocks=i(1, 2),
                free_count=i(2), block_size=16, rows=1)
    append_blocks(**good)

    def bad(error, match, **kw):
        with pytest.raises(error, match=match):
            append_blocks(**{**good, **kw})

    bad(RuntimeError, "ROCm GPU", lens=i(1).cpu())
    bad(ValueError, "new_lens on cpu", new_lens=i(1).cpu())
    bad(TypeError, "int32", new_lens=i(1).long())
    bad(ValueError, "offsets", offsets=i(0, 1, 1))
    bad(ValueError, "block_tables", block_tables=i(0, 1))
    bad(ValueError, "block_tables", block_tables=_i32([[0], [1]], gpu))
    bad(ValueError, "free_count", free_count=i(1, 1))
    bad(ValueError, "block_size", block_size=0)
    bad(ValueError, "rows", rows=-1)
    bad(ValueError, "index", index=i(0, 0))
    many = torch.zeros(4097, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="4096"):
        append_blocks(many, many, torch.zeros(4098, dtype=torch.int32, device=gpu), many.view(-1, 1), i(1), i(0), 16, 0)
    with pytest.raises(ValueError, match="keep"):
        truncate_blocks(i(1), i(1, 2), _i32([[0]], gpu), i(1), i(0), 16)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=gpu)
    k, s = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    for error, match, args in [
            (TypeError, "bf16 or fp16", (k.float(), k.float(), c.float(), c.float(), s)),
            (TypeError, "cache's dtype", (k.half(), k, c, c, s)), (ValueError, "must be", (k[:2], k, c, c, s)),
            (ValueError, "must be", (k[:, :1], k, c, c, s)), (ValueError, "agree", (k, k, c, c[:1], s)),
            (TypeError, "int64", (k, k, c, c, s.int())), (RuntimeError, "ROCm GPU", (k, k, c.cpu(), c.cpu(), s)),
            (ValueError, "contiguous head_dim", (k, k, c.transpose(2, 3), c.transpose(2, 3), s))]:
        with pytest.raises(error, match=match):
            write_kv(*args)
