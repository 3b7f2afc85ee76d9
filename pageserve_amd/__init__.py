"""pageserve_amd: MI355X (gfx950) INT8 weight-only linear path.

A drop-in for pageserve's ``engine/quantization.py``: the same Python API,
computed by hand-written HIP kernels behind a C ABI
(``include/pageserve_amd.h``).
"""

from .cache4 import KVCache4, read_kv4, write_kv4  # noqa: F401
from .paged import append_blocks, tree_attention, truncate_blocks, write_kv  # noqa: F401
from .quantization import (  # noqa: F401
    QuantizedWeight,
    W8A16Weight,
    apply_rope,
    dequantize,
    linear,
    linear_argmax,
    linear_group,
    load_quantized,
    mlp,
    quantize_per_channel,
    rmsnorm,
    rmsnorm_linear_group,
    rmsnorm_mlp,
    rmsnorm_swiglu,
    rope_qk,
    save_quantized,
    swiglu,
)
from .quantization4 import QuantizedWeight4, linear4  # noqa: F401
from .window import accumulate_weights, evict_tokens, window_attention, window_attention4  # noqa: F401

__version__ = "0.1.0"
