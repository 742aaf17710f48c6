from .pools import CacheFull, IndexPool
from .sequence_cache import CODE_DTYPES, PAGE_TOKENS, CacheNeed, LineView, SequenceCache, pages_for

__all__ = ["CODE_DTYPES", "CacheFull", "CacheNeed", "IndexPool", "LineView", "PAGE_TOKENS", "SequenceCache", "pages_for"]
