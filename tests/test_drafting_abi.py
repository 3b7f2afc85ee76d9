"""The C entries of the paged cache and the 4-bit weights: bad arguments are refused on
the host, before any launch (CPU-only)."""

from __future__ import annotations

import ctypes

import pytest

from pageserve_amd import _native

P = ctypes.c_void_p(256)  # a well-aligned address that nothing reads
ODD = ctypes.c_void_p(257)


def _append(lib, lens=P, new=P, tables=P, stride=4, columns=4, free=P, capacity=8, count=P, bs=16, requests=2,
            offsets=P, index=None, rows=5, slots=P, status=P):
    return lib.pgs_append_blocks(lens, new, tables, stride, columns, free, capacity, count, bs, requests, offsets, index,
                                 rows, slots, status, None)


def _truncate(lib, lens=P, keep=P, tables=P, stride=4, columns=4, free=P, capacity=8, count=P, bs=16, requests=2):
    return lib.pgs_truncate_blocks(lens, keep, tables, stride, columns, free, capacity, count, bs, requests, None)


def _cache(**change):
    c = _native.KVCache(k=256, v=256, blocks=4, block_size=16, kv_heads=2, head_dim=128, k_block=4096, k_slot=256,
                        k_head=128, v_block=4096, v_slot=256, v_head=128)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def _write(lib, k=P, v=P, slots=P, rows=3, cache=None, **change):
    c = _cache(**change)
    return lib.pgs_write_kv(k, 256, 128, v, 256, 128, ctypes.byref(c) if cache is None else cache, slots, rows, None)


def _attend(lib, cache=None, workspace=P, given=1 << 40, **change):
    c = _cache(**(cache or {}))
    a = _native.TreeAttentionArgs(q=256, k=256, v=256, out=256, q_row=2048, q_head=128, k_row=256, k_head=128, v_row=256,
                                  v_head=128, out_row=2048, out_head=128, cache=ctypes.pointer(c), block_tables=256,
                                  table_stride=4, columns=4, lens=256, offsets=256, parents=256, rows=5, requests=2,
                                  q_heads=16, max_tokens=64, max_context=64, scale=0.1, dtype=_native.DTYPE_BF16)
    for name, value in change.items():
        setattr(a, name, value)
    return lib.pgs_tree_attention(ctypes.byref(a), workspace, given, None)


def _linear(lib, x=P, qp=P, sp=P, bias=None, res=None, y=P, dtype=1, m=2, n=32, k=64, group=32, ws=None, given=0):
    return lib.pgs_w4a16_linear(x, qp, sp, bias, res, y, dtype, m, n, k, group, ws, given, None)


CASES = [
    (_append, {"requests": -1}), (_append, {"requests": 4097}), (_append, {"bs": 0}), (_append, {"stride": 3}),
    (_append, {"rows": -1}), (_append, {"lens": None}), (_append, {"tables": ODD}), (_append, {"slots": ODD}),
    (_append, {"status": None}), (_append, {"capacity": -1}),
    (_truncate, {"requests": -1}), (_truncate, {"keep": None}), (_truncate, {"bs": -16}), (_truncate, {"count": ODD}),
    (_write, {"rows": -1}), (_write, {"k": None}), (_write, {"v": ODD}), (_write, {"slots": ODD}), (_write, {"blocks": -1}),
    (_write, {"head_dim": 0}), (_write, {"k_slot": -1}),
    (_attend, {"dtype": 0}), (_attend, {"max_tokens": 65}), (_attend, {"max_tokens": 0}), (_attend, {"q_heads": 15}),
    (_attend, {"rows": -1}), (_attend, {"q": None}), (_attend, {"q": 264}), (_attend, {"q_row": 2047}),
    (_attend, {"scale": float("nan")}), (_attend, {"table_stride": 3}), (_attend, {"columns": 1 << 40, "table_stride": 1 << 40}),
    (_attend, {"columns": (1 << 27) - 1, "table_stride": 1 << 27}), (_attend, {"columns": 1 << 62, "table_stride": 1 << 62}),
    (_attend, {"lens": 258}), (_attend, {"workspace": None}), (_attend, {"given": 8}),
    (_attend, {"workspace": ctypes.c_void_p(128)}),
    (_attend, {"cache": {"head_dim": 96}}), (_attend, {"cache": {"block_size": 24}}), (_attend, {"cache": {"k": 0}}),
    (_attend, {"cache": {"kv_heads": 0}}), (_attend, {"cache": {"k_slot": 1 << 30}}), (_attend, {"cache": {"blocks": 0}}),
    (_linear, {"m": -1}), (_linear, {"group": 48}), (_linear, {"k": 40}), (_linear, {"k": 1 << 40}), (_linear, {"dtype": 2}),
    (_linear, {"x": None}), (_linear, {"qp": ODD}), (_linear, {"y": None}), (_linear, {"m": 1 << 40}),
    (_linear, {"n": 1 << 40}), (_linear, {"m": 16, "n": 2048, "k": 11008}),
    (_linear, {"m": 16, "n": 2048, "k": 11008, "ws": P, "given": 64}),
    (_linear, {"m": 16, "n": 2048, "k": 11008, "ws": ctypes.c_void_p(264), "given": 1 << 40}),
]


@pytest.mark.parametrize("call,change", CASES, ids=[f"{f.__name__[1:]}-{'-'.join(map(str, c))}-{i}"
                                                   for i, (f, c) in enumerate(CASES)])
def test_bad_arguments(native_lib, call, change):
    assert call(native_lib, **change) in (1, 2)
    assert native_lib.pgs_last_error()


def test_nothing_to_do(native_lib):
    assert _append(native_lib, requests=0, rows=0) == 0
    assert _truncate(native_lib, requests=0) == 0
    assert _write(native_lib, rows=0) == 0
    assert _attend(native_lib, rows=0) == 0 and _attend(native_lib, requests=0) == 0
    assert _linear(native_lib, m=0) == 0 and _linear(native_lib, n=0) == 0


def test_no_device_is_an_error_not_a_launch(native_lib):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the device check passes there")
    for call in (_append, _truncate, _write, _attend, _linear):
        assert call(native_lib) == 4, call.__name__


def test_workspace_sizes(native_lib):
    f = native_lib.pgs_w4a16_workspace_bytes
    assert f(1, 2048, 2048) == f(0, 2048, 11008) == f(-1, 5, 16) == 0
    for m in (9, 30, 60, 128):
        n = f(m, 2048, 11008)
        assert n % (4 * m * 2048) == 0 and 2 <= n // (4 * m * 2048) <= 8
    g = native_lib.pgs_tree_attention_workspace_bytes
    assert g(5, 5, 16, 2, 128, 1, 100) == 0           # short contexts: one part
    assert g(1, 1, 16, 2, 128, 1, 32768) % (16 * 130 * 4) == 0 != g(1, 1, 16, 2, 128, 1, 32768)
    assert g(64, 1, 16, 2, 128, 64, 100) > 0
    assert g(-1, 1, 16, 2, 128, 1, 100) == g(1, 1, 15, 2, 128, 1, 100) == g(1, 1, 16, 2, 96, 1, 100) == 0
