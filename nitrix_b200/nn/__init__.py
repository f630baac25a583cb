"""``nitrix.nn``-shaped namespace: the attention entry point and its siblings, LayerNorm and the selective scan, and the
operators of a decoder's attention layer: rotary positions, packed sequences, a paged cache and the attention that reads it."""
from .attention import default_scale, qk_rms_norm, scaled_dot_product_attention
from .cache import PagedCache, cache_append, cache_compact, cache_fork, cache_free, decode_attention, paged_cache
from .norm import layer_norm
from .packed import packed_attention
from .rotary import rotary_embedding, rotary_frequencies
from .ssm import selective_scan

__all__ = ["scaled_dot_product_attention", "default_scale", "qk_rms_norm", "layer_norm", "selective_scan", "rotary_embedding",
           "rotary_frequencies", "packed_attention", "PagedCache", "paged_cache", "cache_append", "cache_fork", "cache_free",
           "cache_compact", "decode_attention"]
