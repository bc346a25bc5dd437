from .diffcache import DiffCache
from .mxcache import MxCache
from .pagedcache import PagedCache

__all__ = ["DiffCache", "MxCache", "PagedCache"]
