from .diffcache import DiffCache
from .mxcache import MxCache

__all__ = ["DiffCache", "MxCache"]
