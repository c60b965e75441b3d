from .manager import FREED, CacheError, CacheManager, GroupSpec, PageAllocator, RequestCache, SlotAllocator, TokenBudget

__all__ = ["FREED", "CacheError", "CacheManager", "GroupSpec", "PageAllocator", "RequestCache", "SlotAllocator", "TokenBudget"]
