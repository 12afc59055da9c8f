"""mlxq — MI355X (gfx950) group-wise affine Q4/Q8 quantized linear.

Drop-in for mlx-gen's quantized-linear path: the op triple ``quantize`` / ``dequantize`` /
``quantized_matmul`` (mlx_rs::ops as called from the reference's src/quant.rs and
src/adapters.rs) and the ``QuantizedLinear`` / ``AdaptableLinear`` layer surface built on it; with it, the
operators between a decoder's projections when it serves from a paged key/value cache (paged.py), and a
decoder block's norms, routing and products in microscaled types (mx.py).
All compute runs in libmlxq_hip.so (hand-written HIP for gfx950) through its C ABI.
"""
from ._lib import (MLXQ_ACT_GELU, MLXQ_ACT_GELU_EXACT, MLXQ_ACT_GELU_TANH, MLXQ_ACT_NONE,
                   MLXQ_BFLOAT16, MLXQ_FLOAT16, MLXQ_FLOAT32, MlxqError, LIB_PATH, load)
from .ops import (DEFAULT_GROUP_SIZE, dequantize, embedding, linear, linear_out_dtype,
                  linear_workspace_size, lokr_residual, lora_residual, packed_bits, promote, qmm, qmm_experts, qmv,
                  qmv_valu, quantize, quantize_batched, quantized_matmul, swiglu)
from .nn import (Adapter, AdaptableLinear, LokrAdapter, QuantizedLinear, StackedExperts, TokenEmbedding,
                 has_packed_experts, lin, load_packed_experts, quantize_map)
from .paged import (CacheBatch, PagedCache, cache_append, cache_shapes, cache_tokens, copy_pages, paged_attention, rotary,
                    rotary_frequencies, rotary_table)
from .mx import (Mx, Routing, mx_dequantize, mx_experts, mx_matmul, mx_quantize, rms_norm, rms_norm_backward, route_experts,
                 route_experts_backward, route_plan)
from . import io

__all__ = [
    "MLXQ_ACT_GELU", "MLXQ_ACT_GELU_EXACT", "MLXQ_ACT_GELU_TANH", "MLXQ_ACT_NONE", "MLXQ_BFLOAT16",
    "MLXQ_FLOAT16", "MLXQ_FLOAT32", "MlxqError", "LIB_PATH", "load", "DEFAULT_GROUP_SIZE", "dequantize", "embedding",
    "linear", "linear_out_dtype", "linear_workspace_size", "lokr_residual", "lora_residual", "packed_bits", "promote",
    "qmm", "qmm_experts", "qmv", "qmv_valu", "quantize", "quantize_batched",
    "quantized_matmul", "swiglu", "Adapter", "AdaptableLinear", "LokrAdapter", "QuantizedLinear", "StackedExperts",
    "TokenEmbedding", "has_packed_experts", "lin", "load_packed_experts", "quantize_map", "CacheBatch", "PagedCache", "cache_append",
    "cache_shapes", "cache_tokens", "copy_pages", "paged_attention", "rotary", "rotary_frequencies", "rotary_table",
    "Mx", "Routing", "mx_dequantize", "mx_experts", "mx_matmul", "mx_quantize", "rms_norm", "rms_norm_backward", "route_experts",
    "route_experts_backward", "route_plan", "io",
]
