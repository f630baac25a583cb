"""``nitrix.nn``-shaped namespace: the attention entry point and its siblings, LayerNorm and the selective scan, and the
operators of a decoder layer: the root-mean-square norm, rotary positions, packed sequences, a paged cache (also in 4 or 8 bits)
and the attention that reads it."""
from .attention import default_scale, qk_rms_norm, scaled_dot_product_attention
from .cache import (PagedCache, QuantizedCache, cache_append, cache_compact, cache_fork, cache_free, cache_read, decode_attention,
                    paged_cache, quantized_cache)
from .norm import layer_norm, rms_norm, rms_norm_quantized
from .packed import packed_attention
from .rotary import rotary_embedding, rotary_frequencies
from .ssm import selective_scan

__all__ = ["scaled_dot_product_attention", "default_scale", "qk_rms_norm", "layer_norm", "rms_norm", "rms_norm_quantized",
           "selective_scan", "rotary_embedding", "rotary_frequencies", "packed_attention", "PagedCache", "paged_cache",
           "QuantizedCache", "quantized_cache", "cache_append", "cache_fork", "cache_free", "cache_compact", "cache_read",
           "decode_attention"]
