from .spec import CompositeSpec, PagedKVSpec, StateSpec, leaf_specs
from .manager import (CacheManager, PagePool, SlotPool, CacheError, OutOfPages, OutOfSlots, RELEASED)
from .kv4 import Kv4Cache
from .shared import SharedCache

__all__ = ["Kv4Cache", "SharedCache", "PagedKVSpec", "StateSpec", "CompositeSpec", "leaf_specs", "CacheManager", "PagePool", "SlotPool", "CacheError", "OutOfPages",
           "OutOfSlots", "RELEASED"]
