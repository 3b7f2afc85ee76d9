"""The C entries of the operators of long texts at the sizes that one launch bounds (CPU-only)."""

from __future__ import annotations

import pytest
from test_window_abi import _attend, _read, _write

MOST = (1 << 34) - 1024  # numbers of a call: threads of a launch are fewer than 2^32, each of four numbers at least


@pytest.mark.parametrize("call", [_write, _read])
@pytest.mark.parametrize("heads,dim", [(2, 128), (1, 64), (3, 128), (4096, 64)])
def test_rows_of_a_4_bit_cache(native_lib, call, heads, dim):
    import torch

    most = MOST // (heads * dim)
    size = {"kv_heads": heads, "head_dim": dim}
    assert call(native_lib, rows=most + 1, cache4=size) == 1  # PGS_ERR_INVALID_ARGUMENT
    if not torch.cuda.is_available():  # (a GPU would run them, on these addresses)
        assert call(native_lib, rows=most, cache4=size) == 4  # PGS_ERR_NO_DEVICE: as large as that they are well-formed


@pytest.mark.parametrize("sizes", [{"rows": 8192, "requests": 8192, "max_tokens": 8192, "q_heads": 16},
                                   {"rows": 1 << 16, "requests": 256, "max_tokens": 1 << 16, "q_heads": 64},
                                   {"rows": 1 << 20, "requests": 1 << 20, "max_tokens": 1, "q_heads": 14}])
def test_batches_of_many_requests_and_rows(native_lib, sizes):
    """max_tokens left at its default, the batch's rows, is no reason to refuse a batch"""
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU would run them, on these addresses")
    assert _attend(native_lib, **sizes) == 4  # PGS_ERR_NO_DEVICE: well-formed
    assert _attend(native_lib, **(sizes | {"requests": 1 << 24})) == 1
