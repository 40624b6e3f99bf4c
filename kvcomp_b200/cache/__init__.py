"""Cache classes: the reference's interfaces (models/cache/), and the paged cache of a serving batch."""
from .kvcomp_cache import KVCompCache
from .kvcomp_encode import KVCompCtx
from .paged import PagedKVCache
from ..utils.config import KVCompCacheConfig, KVCompCacheConfigStatic

__all__ = ["KVCompCache", "KVCompCtx", "PagedKVCache", "KVCompCacheConfig", "KVCompCacheConfigStatic"]
