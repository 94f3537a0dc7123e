"""Quantized linear layers with the constructor arguments, parameter names and argument
marshalling of torch_npu.contrib.module.{LinearQuant, LinearA8W8Quant, LinearWeightQuant}, and the
key-value cache that stands between them in a decode step."""
from .linear_quant import LinearQuant, LinearA8W8Quant
from .linear_weight_quant import LinearWeightQuant
from .paged_kv_cache import PagedKVCache

__all__ = ["LinearQuant", "LinearA8W8Quant", "LinearWeightQuant", "PagedKVCache"]
