"""Runtime: packed weight container, decode state and the CUDA kernel layer."""
from .history import TokenHistory
from .kvcache import QuantizedKVCache
from .store import PackedModelStore, PackedWeight

__all__ = ["PackedModelStore", "PackedWeight", "QuantizedKVCache", "TokenHistory"]
