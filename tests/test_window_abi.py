"""The C entries of the operators of long texts: bad arguments are refused on the host,
before any launch (CPU-only)."""

from __future__ import annotations

import ctypes

import pytest

from pageserve_amd import _native

P = ctypes.c_void_p(256)  # a well-aligned address that nothing reads
ODD = ctypes.c_void_p(257)
BIG = 1 << 40


def _set(s, change):
    for name, value in change.items():
        setattr(s, name, value)
    return s


def _cache(change=None):
    c = _native.KVCache(k=256, v=256, blocks=4, block_size=16, kv_heads=2, head_dim=128, k_block=4096, k_slot=256,
                        k_head=128, v_block=4096, v_slot=256, v_head=128)
    return _set(c, change or {})


def _cache4(change=None):
    c = _native.KVCache4(k=256, k_scale=256, v=256, v_scale=256, blocks=4, block_size=16, kv_heads=2, head_dim=128)
    return _set(c, change or {})


def _paged(args, cache, cache4, change):
    if cache is not None:
        args.cache = ctypes.pointer(_cache(cache))
    if cache4 is not None:
        args.cache4 = ctypes.pointer(_cache4(cache4))
    return _set(args, change)


def _attend(lib, cache={}, cache4=None, workspace=P, given=BIG, **change):  # noqa: B006
    a = _native.WindowAttentionArgs(q=256, out=256, lse=256, q_row=2048, q_head=128, out_row=2048, out_head=128,
                                    block_tables=256, table_stride=4, columns=4, lens=256, offsets=256, rows=5, requests=2,
                                    q_heads=16, max_tokens=5, max_context=64, window=8, sinks=4, scale=0.1, dtype=1)
    return lib.pgs_window_attention(ctypes.byref(_paged(a, cache, cache4, change)), workspace, given, None)


def _weigh(lib, cache={}, cache4=None, workspace=P, given=BIG, **change):  # noqa: B006
    a = _native.AccumulateWeightsArgs(q=256, q_row=2048, q_head=128, block_tables=256, table_stride=4, columns=4, lens=256,
                                      offsets=256, lse=256, new_lens=256, weights=256, rows=5, requests=2, q_heads=16,
                                      max_tokens=5, max_context=64, window=8, sinks=4, scale=0.1, dtype=1)
    return lib.pgs_accumulate_weights(ctypes.byref(_paged(a, cache, cache4, change)), workspace, given, None)


def _write(lib, k=P, v=P, k_row=256, v_head=128, dtype=1, cache4={}, slots=P, rows=3):  # noqa: B006
    c = None if cache4 is None else ctypes.byref(_cache4(cache4))
    return lib.pgs_write_kv4(k, k_row, 128, v, 256, v_head, dtype, c, slots, rows, None)


def _read(lib, cache4={}, slots=P, rows=3, k=P, v=P, dtype=1):  # noqa: B006
    c = None if cache4 is None else ctypes.byref(_cache4(cache4))
    return lib.pgs_read_kv4(c, slots, rows, k, v, dtype, None)


def _evict(lib, weights=P, lens=P, budget=P, tables=P, stride=4, columns=4, blocks=4, size=16, requests=2, sinks=0, recent=0,
           context=64, caches=({}, {}), caches4=({},), kept=P, workspace=P, given=BIG):
    c = (_native.KVCache * 2)(*(_cache(x) for x in caches)) if caches else None
    c4 = (_native.KVCache4 * 1)(*(_cache4(x) for x in caches4)) if caches4 else None
    return lib.pgs_evict_tokens(weights, lens, budget, tables, stride, columns, blocks, size, requests, sinks, recent, context,
                                c, 2, c4, 1, kept, workspace, given, None)


SHARED = [{"dtype": 0}, {"rows": -1}, {"requests": -1}, {"q_heads": 15}, {"q_heads": 8192}, {"q_heads": 1}, {"max_tokens": 0},
          {"max_tokens": BIG}, {"max_context": -1}, {"max_context": BIG}, {"window": 0}, {"window": -3}, {"window": BIG},
          {"sinks": -1}, {"sinks": BIG}, {"scale": float("nan")}, {"q": None}, {"q": 264}, {"q_row": 2047}, {"q_head": -8},
          {"lens": None}, {"lens": 258}, {"offsets": None}, {"block_tables": None}, {"block_tables": 258}, {"table_stride": 3},
          {"columns": -1}, {"columns": BIG, "table_stride": BIG}, {"columns": 1 << 62, "table_stride": 1 << 62},
          {"cache": None}, {"cache4": {}}, {"rows": BIG}, {"requests": BIG}]
CACHE = [{"head_dim": 96}, {"block_size": 24}, {"block_size": 0}, {"block_size": 1 << 20}, {"blocks": 0}, {"blocks": BIG},
         {"kv_heads": 0}, {"kv_heads": 5}, {"k": 0}, {"k": 264}]
CASES = (
    [(f, c) for f in (_attend, _weigh) for c in SHARED + [{"cache": x} for x in CACHE + [{"k_slot": 1 << 30}, {"k_head": 12},
                                                                                       {"k_block": -8}]]
     + [{"cache": None, "cache4": x} for x in CACHE + [{"k_scale": 0}, {"k_scale": 258}]]]
    + [(_attend, c) for c in ({"out": None}, {"out": 264}, {"out_row": 4}, {"lse": 258}, {"cache": {"v": 0}},
                              {"cache": {"v_slot": 1 << 30}}, {"cache": {"v_head": 4}}, {"cache": None, "cache4": {"v": 0}},
                              {"cache": None, "cache4": {"v_scale": 264}})]
    + [(_attend, {"rows": 2, "requests": 1, "max_context": 1 << 20, **c}) for c in (
        {"workspace": None, "window": 1 << 20}, {"given": 8, "window": 1 << 20},
        {"workspace": ctypes.c_void_p(128), "window": 1 << 20})]
    + [(_attend, {"rows": 262143, "max_tokens": 262143, "requests": 1, "q_heads": 4096, "cache": {"kv_heads": 1},
                  "columns": 0x7FFF0000 // 16, "table_stride": 0x7FFF0000 // 16, "max_context": 0x7FFFFFFF})]
    + [(_weigh, c) for c in ({"lse": None}, {"lse": 258}, {"weights": None}, {"weights": 258}, {"new_lens": 257})]
    + [(_weigh, {"rows": 200, "max_tokens": 200, **c}) for c in ({"workspace": None}, {"given": 8},
                                                                 {"workspace": ctypes.c_void_p(258)})]
    + [(_write, c) for c in ({"k": None}, {"v": None}, {"slots": None}, {"k": ODD}, {"v": ctypes.c_void_p(264)}, {"slots": ODD},
                             {"k_row": 4}, {"v_head": -8}, {"dtype": 0}, {"dtype": 7}, {"rows": -1}, {"rows": BIG},
                             {"cache4": None})]
    + [(_read, c) for c in ({"k": None}, {"v": ODD}, {"slots": ODD}, {"dtype": 3}, {"rows": -1}, {"rows": BIG}, {"cache4": None})]
    + [(f, {"cache4": x}) for f in (_write, _read) for x in CACHE if x not in ({"blocks": 0}, {"kv_heads": 5})]
    + [(_evict, c) for c in ({"weights": None}, {"weights": ODD}, {"lens": None}, {"budget": ODD}, {"tables": None}, {"kept": None},
                             {"kept": ODD}, {"stride": 3}, {"columns": -1}, {"columns": BIG, "stride": BIG}, {"blocks": -1},
                             {"blocks": 5}, {"size": 8}, {"size": 24}, {"size": 32}, {"requests": -1}, {"requests": BIG},
                             {"sinks": -1}, {"sinks": BIG}, {"recent": -1}, {"recent": BIG}, {"context": -1}, {"context": BIG},
                             {"workspace": None}, {"given": 16}, {"workspace": ODD}, {"caches": None}, {"caches4": None},
                             {"caches": ({}, {"k": 0})}, {"caches": ({}, {"v": 257})}, {"caches": ({}, {"k_slot": -8})},
                             {"caches": ({}, {"head_dim": 64})}, {"caches": ({"kv_heads": 1}, {})},
                             {"caches4": ({"head_dim": 96},)}, {"caches4": ({"v_scale": 0},)}, {"caches4": ({"k": 264},)},
                             {"requests": 65536, "caches": ({"kv_heads": 4096}, {"kv_heads": 4096})})]
)


@pytest.mark.parametrize("call,change", CASES, ids=[f"{f.__name__[1:]}-{'-'.join(map(str, c))}-{i}"
                                                   for i, (f, c) in enumerate(CASES)])
def test_bad_arguments(native_lib, call, change):
    assert call(native_lib, **change) in (1, 2)


def test_null_arguments(native_lib):
    assert native_lib.pgs_window_attention(None, P, BIG, None) in (1, 2)
    assert native_lib.pgs_accumulate_weights(None, P, BIG, None) in (1, 2)


@pytest.mark.parametrize("call", [_attend, _weigh, _write, _read, _evict])
def test_well_formed_calls_need_a_gpu(native_lib, call):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU would run them, on these addresses")
    assert call(native_lib) == 4  # PGS_ERR_NO_DEVICE


def test_nothing_to_do(native_lib):
    assert _attend(native_lib, rows=0) == 0 and _attend(native_lib, requests=0) == 0
    assert _weigh(native_lib, requests=0) == 0
    assert _write(native_lib, rows=0) == 0 and _read(native_lib, rows=0) == 0
    assert _evict(native_lib, requests=0) == 0


def test_workspaces(native_lib):
    def need(four=False, columns=6250, **change):
        c, c4 = _cache(), _cache4()
        a = _native.WindowAttentionArgs(rows=1, requests=1, q_heads=16, max_tokens=1, max_context=64, window=1 << 30,
                                        columns=columns, table_stride=columns)
        if four:
            a.cache4 = ctypes.pointer(c4)
        else:
            a.cache = ctypes.pointer(c)
        return native_lib.pgs_window_attention_workspace_bytes(ctypes.byref(_set(a, change)))

    assert need() == need(four=True) == 0
    assert need(max_context=100000) > 0
    # a window bounds the split whatever the context, and no request has more rows than the batch
    assert need(max_context=100000, window=100, sinks=4) == 0
    assert need(max_context=100000) == need(max_context=100000, max_tokens=500)
    many = {"rows": 900, "max_tokens": 900, "max_context": 100000}
    assert need(**many) > 0
    # (many rows over a 4-bit cache: one request's tokens in 16 bits, and the table of them)
    assert need(four=True, **many) - need(**many) == 6250 * (2 * 64 * 128 + 4)
    assert need(rows=-1) == need(q_heads=15) == need(columns=-1) == 0
    assert native_lib.pgs_window_attention_workspace_bytes(None) == 0
    assert native_lib.pgs_evict_tokens_workspace_bytes(3, 100) == 3 * 101 * 4
    assert native_lib.pgs_evict_tokens_workspace_bytes(0, 100) == 0
