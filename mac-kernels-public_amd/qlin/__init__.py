"""qlin: packed-weight quantized linear ops for AMD MI355X (gfx950).

Drop-in for comfy-kitchen's packed-weight linear family (roblennon/mac-kernels-public): INT8 with
ConvRot rotation (weight-only, fp16 MFMA), W4A8 / W6A8 (AsymW4A8Int8 storage, int8 MFMA on
per-token int8 activations) and the GGUF block formats Q4_0..Q6_K, IQ4_NL, IQ4_XS (weight-only,
decoded inside the kernels).  Between a block's packed linears: rotation by positions on several axes,
per-head norms of q and k with it (forward, backward, into a paged cache), the tables of a step
over that cache and attention of one new token over it.  Everything runs in libqlin.so (HIP, C ABI in include/qlin.h).
"""
from .attention import (
    PagedPlan,
    axis_rope,
    axis_rope_trainable,
    paged_attention,
    paged_plan,
    qk_norm_rope,
    qk_norm_rope_grad,
    qk_norm_rope_store,
    qk_norm_rope_trainable,
    rope_frequencies,
)
from .autograd import int8_linear_grad_input, int8_linear_trainable, w4a8_linear_grad_input, w4a8_linear_trainable
from .exceptions import NoCapableBackendError, QlinError
from .gguf import GGUF_TYPES, gguf_type_id
from .layouts import AsymW4A8Int8Layout, QuantizedTensor, TensorWiseINT8Layout
from .loader import PackedLinear, gguf_header, load_gguf, load_safetensors, quantized_linears, safetensors_header
from .ops import (
    dequantize_gguf,
    dequantize_int8,
    dequantize_int8_convrot_weight,
    dequantize_w4a8_int8_weight,
    gguf_linear,
    int8_linear,
    quantize_int8_rowwise,
    w4a8_int8_grid,
    w4a8_int8_linear,
)
from .registry import registry

__all__ = [
    "NoCapableBackendError", "QlinError", "GGUF_TYPES", "gguf_type_id", "dequantize_gguf", "dequantize_int8",
    "dequantize_int8_convrot_weight", "dequantize_w4a8_int8_weight", "gguf_linear", "int8_linear",
    "quantize_int8_rowwise", "w4a8_int8_grid", "w4a8_int8_linear", "registry", "PackedLinear", "gguf_header",
    "load_gguf", "load_safetensors", "quantized_linears", "safetensors_header", "int8_linear_grad_input",
    "int8_linear_trainable", "w4a8_linear_grad_input", "w4a8_linear_trainable", "AsymW4A8Int8Layout",
    "QuantizedTensor", "TensorWiseINT8Layout", "PagedPlan", "axis_rope", "axis_rope_trainable", "paged_attention",
    "paged_plan", "qk_norm_rope", "qk_norm_rope_grad", "qk_norm_rope_store", "qk_norm_rope_trainable", "rope_frequencies",
]
