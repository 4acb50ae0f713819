"""models: QuantizedLinear and the gptq::linear operator (the reference's
models/layers.py), and the attention between a decoder layer's quantized
projections (``attention.attention`` keeps its module's name free here); the
reference's model adapters are not part of this path."""
from .attention import (PagedBatch, PagedKVCache, QuantizedAttention, packed_positions, paged_attention, rotary,
                        rotary_append, rotary_frequencies, rotary_table)
from .layers import FusedQuantizedLinear, QuantizedLinear, replace_with_quantized_layers

__all__ = ["FusedQuantizedLinear", "QuantizedLinear", "replace_with_quantized_layers", "PagedBatch", "PagedKVCache",
           "QuantizedAttention", "packed_positions", "paged_attention", "rotary", "rotary_append",
           "rotary_frequencies", "rotary_table"]
