from .cache import KVCache, QuantizedKVCache
from .layers import Attention, Linear, MultiHeadAttention, causal_mask, softmax

__all__ = ["Attention", "KVCache", "Linear", "MultiHeadAttention", "QuantizedKVCache", "causal_mask", "softmax"]
