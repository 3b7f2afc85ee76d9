"""The C entries of the operators of long texts at the sizes that one launch bounds (CPU-only)."""

from __future__ import annotations

import pytest
from test_window_abi import _read, _write

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
