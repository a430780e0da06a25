from .needs import CACHE_KINDS, PAGE, CacheNeed, StateNeed, register_cache_kind
from .pool import CacheFull, FreeList
from .share import PlanCapacity, SharePlan, TileShape, most_part_rows, scratch_rows, share_pays, share_tree
from .store import KVGroup, SequenceCache, pages_for

__all__ = ["PAGE", "CACHE_KINDS", "CacheNeed", "StateNeed", "CacheFull", "FreeList", "KVGroup", "SequenceCache", "pages_for",
           "register_cache_kind", "SharePlan", "PlanCapacity", "TileShape", "share_tree", "share_pays", "most_part_rows", "scratch_rows"]
