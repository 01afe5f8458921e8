"""hexagon_mlir_amd — MI355X-native replacement of Hexagon-MLIR's matmul / GEMV /
RMSNorm / softmax hot path, and the operators of a serving loop around it
(block tables, rotation of queries and keys, key/value caches of 8 and 4 bits,
attention over them, sampling, verification of drafted tokens).

Layers:
  * ``csrc/``      hand-written HIP kernels for gfx950 behind the C ABI of
                   ``include/hxmi.h`` (built into ``lib/libhxmi.so``);
  * ``hxmi``       ctypes binding and torch-tensor ops over that ABI;
  * ``backend``    the reference's Python surface (``HexagonOptions``,
                   ``TorchMLIRHexagonLauncher.run_torch_mlir``) on top of it.

The directory name carries a dash, so it is imported under the module name
``hexagon_mlir_amd`` (see ``load_package`` in the repository's
``__graft_entry__.py``).
"""
from . import hxmi, weights
from .hxmi import (
    HxmiError,
    HxmiNotBuiltError,
    KVCache,
    KVCache4,
    KVPlan,
    Verified,
    attention,
    bgemm,
    fold_rms_weight,
    gemm,
    gemv,
    hexkl_matmul,
    kv_append,
    kv_attention,
    kv_plan,
    kv_read,
    kv_trim,
    linear,
    load_library,
    pack_gate_up,
    qk_rope,
    quantize_int8,
    rms_norm,
    rms_norm_linear,
    rope_frequencies,
    sample,
    set_tuning,
    softmax,
    tuning,
    verify,
    w8a16_linear,
)

__all__ = [
    "hxmi",
    "weights",
    "HxmiError",
    "HxmiNotBuiltError",
    "KVCache",
    "KVCache4",
    "KVPlan",
    "Verified",
    "attention",
    "bgemm",
    "fold_rms_weight",
    "gemm",
    "gemv",
    "hexkl_matmul",
    "kv_append",
    "kv_attention",
    "kv_plan",
    "kv_read",
    "kv_trim",
    "linear",
    "load_library",
    "pack_gate_up",
    "qk_rope",
    "quantize_int8",
    "rms_norm",
    "rms_norm_linear",
    "rope_frequencies",
    "sample",
    "set_tuning",
    "softmax",
    "tuning",
    "verify",
    "w8a16_linear",
]
